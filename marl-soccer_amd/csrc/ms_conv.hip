// ms_conv.hip — short causal convolution over time, per channel, with its gradients (gfx950).
//
//   pre[t] = b + sum_j w[W-1-j] x[t-j],  out = silu(pre) or pre,  j < W <= 4,
// where x[t-j] counts only if no episode starts in (t-j, t], and steps before 0 are the state's.
// Backward, with p[t] = dout[t] act'(pre[t]) and the same condition:
//   dx[t] = sum_j w[W-1-j] p[t+j],  dw[W-1-j] = sum_t p[t] x[t-j],  db = sum_t p[t].
//
// Bound by HBM: one read of x and one write of out (backward: x, dout, dx), a few FMAs a value.
// A thread owns 16 B of neighbouring channels (one 16-B access a step; 8 B backward, where weights,
// windows and sums would take 180 registers at 16 B and halve the waves: 178 -> 160 us for 128 x 2,048
// x 128 f32, forward and backward) and walks a span of steps with its window of W - 1 inputs in
// registers; a span begins by re-reading the W - 1 steps before it, which is what splitting the time
// axis costs. 4 rows of 4,099 steps x 2,048 bf16: 32 us, 4.2 TB/s; 2,048 rows of 128 x 128 f32: forward
// 48 us, 5.6 TB/s, backward 96 us, 4.2 TB/s (403 MB: x, dout, dx).
#include "ms_sequence.h"

thread_local char g_sequence_error[256] = "";

extern "C" const char* ms_sequence_last_error(void) { return g_sequence_error; }

namespace conv {
using namespace seq;

constexpr int THREADS = 256;

struct Shape {  // the launch: a block covers `cols` groups of E channels and `slots` spans at a time
  int cols_log2;
  int64_t groups, spans, span, items, blocks_c, blocks_p;
};

// Every access is E aligned channels, so the loads of BATCH steps are issued together without a branch
// between them. A block takes items (a row's span) in turn: many rows of one step read their weights once.
constexpr int BATCH = 4;
template <typename T, int E, int W>
__global__ __launch_bounds__(THREADS) void forward(const ms_conv_io io, const Shape sh) {
  const int cols = 1 << sh.cols_log2, slots = THREADS >> sh.cols_log2;
  const int64_t bc = blockIdx.x % sh.blocks_c, bp = blockIdx.x / sh.blocks_c;
  const int64_t group = bc * cols + (threadIdx.x & (cols - 1)), c = group * E, D = io.channels;
  if (group >= sh.groups) return;
  float w[W][E], b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    b[e] = io.bias ? io.bias[c + e] : 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = io.weight[(c + e) * W + k];
  }
  for (int64_t item = bp * slots + (threadIdx.x >> sh.cols_log2); item < sh.items; item += sh.blocks_p * slots) {
    const int64_t span = sh.spans > 1 ? item / io.rows : 0, r = item - span * io.rows, t0 = span * sh.span;
    const int64_t t1 = t0 + sh.span < io.steps ? t0 + sh.span : io.steps;
    const T* x = (const T*)io.x + r * io.x_r + c;
    T* out = (T*)io.out + r * io.out_r + c;
    const uint8_t* starts = io.starts ? io.starts + r * io.starts_r : nullptr;
    const T* state = io.state ? (const T*)io.state + r * (W - 1) * D + c : nullptr;
    float win[W - 1][E];  // win[k]: the input W - 1 - k steps back
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      const int64_t t = t0 - (W - 1) + k;
      typename Vec<T, E>::type v;
      if (t >= 0) {
        v = load<T, E>(x + t * io.x_t);
        if (starts && starts[t * io.starts_t]) {
#pragma unroll
          for (int j = 0; j < k; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) win[j][e] = 0.0f;
        }
      } else if (state) {
        v = load<T, E>(state + (W - 1 + t) * D);
      } else {
        v = 0;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) win[k][e] = (float)v[e];
    }
    const T* px = x + t0 * io.x_t;
    T* po = out + t0 * io.out_t;
    const uint8_t* ps = starts ? starts + t0 * io.starts_t : nullptr;
    const bool act = io.silu;
    auto step = [&](const typename Vec<T, E>::type& v, bool cut) __attribute__((always_inline)) {
      if (cut) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e) win[j][e] = 0.0f;
      }
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float a = b[e];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) a = __builtin_fmaf(w[k][e], win[k][e], a);
        a = __builtin_fmaf(w[W - 1][e], (float)v[e], a);
        y[e] = act ? silu(a) : a;
#pragma unroll
        for (int k = 0; k < W - 2; ++k) win[k][e] = win[k + 1][e];
        win[W - 2][e] = (float)v[e];
      }
      store<T, E>(po, y);
      po += io.out_t;
    };
    int64_t t = t0;
    for (; t + BATCH <= t1; t += BATCH) {
      typename Vec<T, E>::type v[BATCH];
      bool cut[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        v[k] = load<T, E>(px);
        px += io.x_t;
        cut[k] = ps && ps[k * io.starts_t];
      }
      if (ps) ps += BATCH * io.starts_t;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) step(v[k], cut[k]);
    }
    for (; t < t1; ++t) {
      const typename Vec<T, E>::type v = load<T, E>(px);
      px += io.x_t;
      step(v, ps && ps[0]);
      if (ps) ps += io.starts_t;
    }
    if (io.new_state && t1 == io.steps) {
      T* ns = (T*)io.new_state + r * (W - 1) * D + c;
#pragma unroll
      for (int k = 0; k < W - 1; ++k) store<T, E>(ns + k * D, win[k]);
    }
  }
}

// p[t] reaches dx of steps t - W + 1 .. t: pend[j] collects dx[t - j], complete (and stored) when it
// falls out of the window. reach: how many steps back belong to step t's episode. A span stores the
// steps of its own and runs W - 1 steps past them, whose p counts for dx but not for dw and db. FULL: rows
// are aligned for E channels; otherwise the same threads move them one by one, so that no sum changes.
template <typename T, int E, int W, bool FULL>
__global__ __launch_bounds__(THREADS) void backward(const ms_conv_io io, const Shape sh, float* __restrict__ parts) {
  __shared__ float red[THREADS];
  const int cols = 1 << sh.cols_log2, slots = THREADS >> sh.cols_log2;
  const int64_t bc = blockIdx.x % sh.blocks_c, bp = blockIdx.x / sh.blocks_c;
  const int col = threadIdx.x & (cols - 1), slot = threadIdx.x >> sh.cols_log2;
  const int64_t group = bc * cols + col, D = io.channels, c = group * E;
  const bool some = group < sh.groups;
  float w[W][E], b[E], dw[W][E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    b[e] = io.bias && some ? io.bias[c + e] : 0.0f;
    db[e] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k][e] = some ? io.weight[(c + e) * W + k] : 0.0f;
      dw[k][e] = 0.0f;
    }
  }
  for (int64_t item = bp * slots + slot; some && item < sh.items; item += sh.blocks_p * slots) {
    const int64_t r = item % io.rows, t0 = item / io.rows * sh.span;
    const int64_t t1 = t0 + sh.span < io.steps ? t0 + sh.span : io.steps;
    const int64_t t2 = t1 + W - 1 < io.steps ? t1 + W - 1 : io.steps;
    const T* x = (const T*)io.x + r * io.x_r + c;
    const T* dout = (const T*)io.dout + r * io.dout_r + c;
    T* dx = (T*)io.dx + r * io.dx_r + c;
    const uint8_t* starts = io.starts ? io.starts + r * io.starts_r : nullptr;
    const int64_t row = r * (W - 1) * D + c;
    float win[W - 1][E], pend[W - 1][E];  // pend[j]: dx of step t - 1 - j as far as it is known
    int reach = 0;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      const int64_t t = t0 - (W - 1) + k;
      typename Vec<T, E>::type v;
      v = 0;
      reach = reach < W - 1 ? reach + 1 : W - 1;
      if (t >= 0) {
        v = load<T, E>(x + t * io.x_t, E, FULL);
        if (starts && starts[t * io.starts_t]) {
          reach = 0;
#pragma unroll
          for (int j = 0; j < k; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) win[j][e] = 0.0f;
        }
      } else if (io.state) {
        v = load<T, E>((const T*)io.state + row + (W - 1 + t) * D, E, FULL);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        win[k][e] = (float)v[e];
        pend[k][e] = 0.0f;
      }
    }
    const bool act = io.silu;
    // after the W - 1 steps before t0, reach counts how many of the steps t0 - 1, t0 - 2, ... belong
    // to step t0 - 1's episode (that step itself not counted)
    auto flush = [&](int64_t t, const float (&g)[E]) __attribute__((always_inline)) {  // dx[t] is complete
      if (t >= t0 && t < t1) store<T, E>(dx + t * io.dx_t, g, E, FULL);
      if (t < 0 && t0 == 0 && io.dstate) store<T, E>((T*)io.dstate + row + (W - 1 + t) * D, g, E, FULL);
    };
    auto step = [&](int64_t t, const typename Vec<T, E>::type& v, const typename Vec<T, E>::type& d, bool cut) __attribute__((always_inline)) {
      reach = reach < W - 1 ? reach + 1 : W - 1;
      if (cut) {
        reach = 0;
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e) win[j][e] = 0.0f;
      }
      const bool own = t < t1;
      float done[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float a = b[e];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) a = __builtin_fmaf(w[k][e], win[k][e], a);
        a = __builtin_fmaf(w[W - 1][e], (float)v[e], a);
        const float p = act ? (float)d[e] * silu_slope(a) : (float)d[e];
        if (own) {
          db[e] += p;
#pragma unroll
          for (int k = 0; k < W - 1; ++k) dw[k][e] = __builtin_fmaf(p, win[k][e], dw[k][e]);
          dw[W - 1][e] = __builtin_fmaf(p, (float)v[e], dw[W - 1][e]);
        }
#pragma unroll
        for (int j = 1; j < W; ++j)
          if (j <= reach) pend[j - 1][e] = __builtin_fmaf(w[W - 1 - j][e], p, pend[j - 1][e]);
        done[e] = pend[W - 2][e];
#pragma unroll
        for (int j = W - 2; j > 0; --j) pend[j][e] = pend[j - 1][e];
        pend[0][e] = w[W - 1][e] * p;
#pragma unroll
        for (int k = 0; k < W - 2; ++k) win[k][e] = win[k + 1][e];
        win[W - 2][e] = (float)v[e];
      }
      flush(t - (W - 1), done);
    };
    const T* px = x + t0 * io.x_t;
    const T* pd = dout + t0 * io.dout_t;
    const uint8_t* ps = starts ? starts + t0 * io.starts_t : nullptr;
    int64_t t = t0;
    for (; t + BATCH <= t2; t += BATCH) {
      typename Vec<T, E>::type v[BATCH], d[BATCH];
      bool cut[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        v[k] = load<T, E>(px, E, FULL);
        d[k] = load<T, E>(pd, E, FULL);
        px += io.x_t;
        pd += io.dout_t;
        cut[k] = ps && ps[k * io.starts_t];
      }
      if (ps) ps += BATCH * io.starts_t;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) step(t + k, v[k], d[k], cut[k]);
    }
    for (; t < t2; ++t) {
      const typename Vec<T, E>::type v = load<T, E>(px, E, FULL), d = load<T, E>(pd, E, FULL);
      px += io.x_t;
      pd += io.dout_t;
      step(t, v, d, ps && ps[0]);
      if (ps) ps += io.starts_t;
    }
    if (t2 == io.steps) {  // the last steps, and the gradient of the state handed on
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (io.dnew_state && j <= reach) {
          const typename Vec<T, E>::type g = load<T, E>((const T*)io.dnew_state + row + (W - 2 - j) * D, E, FULL);
#pragma unroll
          for (int e = 0; e < E; ++e) pend[j][e] += (float)g[e];
        }
        flush(t2 - 1 - j, pend[j]);
      }
    }
  }
  // the block's sums: slots of the same channels in turn, in a fixed order and in float64 as what follows
  float* to = parts + bp * (W + 1) * D;
#pragma unroll
  for (int k = 0; k <= W; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      __syncthreads();
      red[threadIdx.x] = k < W ? dw[k < W ? k : 0][e] : db[e];
      __syncthreads();
      if (slot == 0 && some) {
        double a = 0.0;
        for (int s = 0; s < slots; ++s) a += red[s * cols + col];
        to[(c + e) * (W + 1) + k] = (float)a;
      }
    }
}

// parts (P, D, W + 1) added up -> dweight (D, W), dbias (D)
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void finish(const float* __restrict__ in, int64_t parts, int64_t D, int W,
                                                     float* __restrict__ dweight, float* __restrict__ dbias) {
  __shared__ double s[WAVES][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float sum = (float)sum_share<WAVES>(in, 0, parts, D * (W + 1), c, s);
  if (threadIdx.x >= 64 || c >= D * (W + 1)) return;
  const int64_t d = c / (W + 1);
  const int k = (int)(c - d * (W + 1));
  if (k < W) {
    if (dweight) dweight[d * W + k] = sum;
  } else if (dbias) {
    dbias[d] = sum;
  }
}

// How the work is cut: spans of steps long enough that the W - 1 re-read steps cost little, short
// enough that there are threads for every SIMD several times over.
constexpr int64_t CHAIN = MS_SUM_CHAIN;  // steps that a thread adds up in float32 for dw and db
Shape shape(const ms_conv_io& io, bool back, int E) {
  Shape s = {};
  s.groups = io.channels / E;
  while ((1 << s.cols_log2) < s.groups && s.cols_log2 < 8) ++s.cols_log2;
  const int64_t slots = THREADS >> s.cols_log2;
  s.blocks_c = (s.groups + (1 << s.cols_log2) - 1) >> s.cols_log2;
  const int64_t want = 262144;  // threads: 256 CUs x 16 waves
  const int64_t have = s.groups * io.rows;
  int64_t spans = have > 0 ? (want + have - 1) / have : 1;
  const int64_t most = (io.steps + 15) / 16;  // 16 steps at least: 3 re-read
  spans = spans > most ? most : spans;
  if (back && spans * CHAIN < io.steps) spans = (io.steps + CHAIN - 1) / CHAIN;
  spans = spans < 1 ? 1 : spans;
  s.span = (io.steps + spans - 1) / spans;
  s.span = s.span < 1 ? 1 : s.span;
  s.spans = io.steps > 0 ? (io.steps + s.span - 1) / s.span : 1;
  s.items = s.spans * io.rows;
  s.blocks_p = (s.items + slots - 1) / slots;
  s.blocks_p = s.blocks_p < 1 ? 1 : s.blocks_p;
  // As many blocks as fill the chip: backward each leaves sums to be added (1,536: 150 us for 2,048 rows of
  // 128 x 128 f32, with 1,024 156), forward each reads its weights. There 16 B a thread leave registers for
  // 1,024 blocks at a time (65,536 rows of one step x 128 bf16: 27 us, 40 uncapped); fewer bytes take four
  // rounds (7,697 x 2,692 f16: 46 us, with 1,024 49, uncapped 52).
  const bool wide = E * (io.dtype == 0 ? 4 : 2) == 16;
  int64_t cap = ((back ? 1536 : wide ? 1024 : 4096) + s.blocks_c - 1) / s.blocks_c;
  if (back) {  // more where a thread's items would be more than CHAIN steps
    const int64_t turn = slots * (CHAIN / s.span > 1 ? CHAIN / s.span : 1), least = (s.items + turn - 1) / turn;
    cap = cap < least ? least : cap;
  }
  if (s.blocks_p > cap) s.blocks_p = cap;
  return s;
}

const char* check(const ms_conv_io* io, bool back) {
  if (!io) return "no arguments";
  if (io->dtype < 0 || io->dtype > 2) return "dtype must be 0 (float32), 1 (bfloat16) or 2 (float16)";
  if (io->width < 2 || io->width > 4) return "width must be 2, 3 or 4";
  if (io->steps < 0 || io->rows < 0 || io->channels <= 0) return "steps and rows must be >= 0, channels > 0";
  if (io->rows > 0 && io->steps > (int64_t)1 << 40) return "too many steps";
  if (!io->weight) return "weight is NULL";
  const bool some = io->steps > 0 && io->rows > 0;
  if (some && !io->x) return "x is NULL";
  if (!back && some && !io->out) return "out is NULL";
  if (!back && io->new_state && io->new_state == io->state && io->steps > 1)
    return "new_state may be the state only for one step";
  if (back && some && (!io->dout || !io->dx)) return "dout or dx is NULL";
  return nullptr;
}

bool rows_aligned(const ms_conv_io& io, bool back, int64_t E) {
  const int64_t elem = io.dtype == 0 ? 4 : 2;
  auto state = [&](const void* p) { return !p || aligned(p, io.channels, 0, elem, E); };
  return aligned(io.x, io.x_t, io.x_r, elem, E) && state(io.state) &&
         (back ? aligned(io.dout, io.dout_t, io.dout_r, elem, E) && aligned(io.dx, io.dx_t, io.dx_r, elem, E) && state(io.dstate) &&
                     state(io.dnew_state)
               : aligned(io.out, io.out_t, io.out_r, elem, E) && state(io.new_state));
}
// Channels a thread: 16 B of them forward, 8 B backward, or as many as divide the channels and, forward,
// keep every access aligned. One by one, neighbouring lanes still read neighbouring values: 7,697 rows of
// a step x 2,692 f16 take 46 us, 413 with 8 channels a thread and guards.
int channels_a_thread(const ms_conv_io& io, bool back) {
  int E = (back ? 8 : 16) / (io.dtype == 0 ? 4 : 2);
  while (E > 1 && (io.channels % E || (!back && !rows_aligned(io, false, E)))) E /= 2;
  return E;
}

template <typename T, int E>
int run_forward(const ms_conv_io& io, hipStream_t stream) {
  const Shape s = shape(io, false, E);
  const int64_t blocks = s.blocks_c * s.blocks_p;
  if (too_many(blocks, THREADS)) return fail(MS_ERR_INVALID_ARGUMENT, "ms_conv_forward", "too large");
  const dim3 grid((unsigned)blocks), block(THREADS);
  switch (io.width) {
    case 2: hipLaunchKernelGGL((forward<T, E, 2>), grid, block, 0, stream, io, s); break;
    case 3: hipLaunchKernelGGL((forward<T, E, 3>), grid, block, 0, stream, io, s); break;
    default: hipLaunchKernelGGL((forward<T, E, 4>), grid, block, 0, stream, io, s); break;
  }
  return launched("ms_conv_forward");
}
template <typename T>
int forward_as(const ms_conv_io& io, hipStream_t stream) {
  const int E = channels_a_thread(io, false);
  if constexpr (sizeof(T) == 2)
    if (E == 8) return run_forward<T, 8>(io, stream);
  if (E == 4) return run_forward<T, 4>(io, stream);
  return E == 2 ? run_forward<T, 2>(io, stream) : run_forward<T, 1>(io, stream);
}
template <typename T, int E, bool FULL>
int run_backward(const ms_conv_io& io, hipStream_t stream) {
  const Shape s = shape(io, true, E);
  const int64_t columns = io.channels * (io.width + 1);
  if (too_many(s.blocks_c * s.blocks_p, THREADS) || too_many((columns + 63) / 64, 1024))
    return fail(MS_ERR_INVALID_ARGUMENT, "ms_conv_backward", "too large");
  const dim3 grid((unsigned)(s.blocks_c * s.blocks_p)), block(THREADS);
  float* parts = (float*)io.workspace;
  switch (io.width) {
    case 2: hipLaunchKernelGGL((backward<T, E, 2, FULL>), grid, block, 0, stream, io, s, parts); break;
    case 3: hipLaunchKernelGGL((backward<T, E, 3, FULL>), grid, block, 0, stream, io, s, parts); break;
    default: hipLaunchKernelGGL((backward<T, E, 4, FULL>), grid, block, 0, stream, io, s, parts); break;
  }
  if (int rc = launched("ms_conv_backward")) return rc;
  if (!io.dweight && !io.dbias) return MS_OK;
  hipLaunchKernelGGL(finish<16>, dim3((unsigned)((columns + 63) / 64)), dim3(1024), 0, stream, parts, s.blocks_p, io.channels,
                     io.width, io.dweight, io.dbias);
  return launched("ms_conv_backward");
}
template <typename T>
int backward_as(const ms_conv_io& io, hipStream_t stream) {
  const int E = channels_a_thread(io, true);
  const bool full = rows_aligned(io, true, E);
  if constexpr (sizeof(T) == 2)
    if (E == 4) return full ? run_backward<T, 4, true>(io, stream) : run_backward<T, 4, false>(io, stream);
  if (E == 2) return full ? run_backward<T, 2, true>(io, stream) : run_backward<T, 2, false>(io, stream);
  return run_backward<T, 1, true>(io, stream);
}

}  // namespace conv

extern "C" {

int ms_conv_forward(const ms_conv_io* io, void* stream) {
  if (const char* why = conv::check(io, false)) return seq::fail(MS_ERR_INVALID_ARGUMENT, "ms_conv_forward", why);
  if (io->rows == 0 || (io->steps == 0 && !io->new_state)) return MS_OK;
  const hipStream_t st = (hipStream_t)stream;
  return io->dtype == 0 ? conv::forward_as<float>(*io, st) : io->dtype == 1 ? conv::forward_as<seq::bf16>(*io, st) : conv::forward_as<seq::f16>(*io, st);
}

int64_t ms_conv_workspace(const ms_conv_io* io) {
  if (conv::check(io, true)) return 0;
  const conv::Shape s = conv::shape(*io, true, conv::channels_a_thread(*io, true));
  return s.blocks_p * io->channels * (io->width + 1) * (int64_t)sizeof(float);
}

int ms_conv_backward(const ms_conv_io* io, void* stream) {
  if (const char* why = conv::check(io, true)) return seq::fail(MS_ERR_INVALID_ARGUMENT, "ms_conv_backward", why);
  if (!io->workspace || ((uintptr_t)io->workspace & 15u) || io->workspace_bytes < ms_conv_workspace(io))
    return seq::fail(MS_ERR_INVALID_ARGUMENT, "ms_conv_backward", "the workspace is missing, misaligned or too small");
  const hipStream_t st = (hipStream_t)stream;
  return io->dtype == 0 ? conv::backward_as<float>(*io, st) : io->dtype == 1 ? conv::backward_as<seq::bf16>(*io, st) : conv::backward_as<seq::f16>(*io, st);
}

}  // extern "C"
