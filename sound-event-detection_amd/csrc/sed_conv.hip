// Causal depthwise convolution along the frames of a clip, with bias and SiLU, its gradient and its one-frame form, gfx950.
//
//   u_t[d] = bias[d] + sum_k w[d,k] x_{t-W+1+k}[d],  y = act(u),  x before the first frame = state (or 0)
//
// Bound: HBM (read x, write y; the gradient reads x and dy and writes dx).  A wave has 64 V neighbouring channels and a run of
// TL frames of one clip: which rows it meets and where they lie is the same for all its lanes (scalar work), a lane keeps the
// window of WM rows, the weights and, in the gradient, the sums of its V channels in registers.  Rows come WM at a time, the
// next WM on their way while WM are worked on.  A row is read once but for the WM - 1 in front of a run (and behind it, in the
// gradient).  WM is W, or 2 for 1 and 8 for 5 to 8.  V = 4 where rows allow it and there are channels enough for a wave (2 in the
// gradient of more than 4 taps), else 1.  The weight gradient is summed per lane over its run, written once per run and added over
// the runs in a fixed order.  Sums are fp32 and every output is rounded once.
//
// Measured (MI355X): 16 x 4096 x 1536 bf16, 4 taps with SiLU: forward 79 us for 403 MB (5.1 TB/s, what a 1 GiB copy reaches),
// gradient 142 us for 604 MB (4.3 TB/s; 150 with a condition at every load, 145 with registers for four waves a vector unit); runs
// of 16 / 32 / 64 frames forward: 84 / 79 / 80 us, of 32 / 64 / 128 in the gradient with its weight sums: 164 / 162 / 167 us at the
// time.  A thread per 8 channels with its own row addresses took 168 and 407 us.
#include "seq_core.h"

#include <algorithm>

namespace sed {
namespace {

struct ConvParams {
  sed_conv_args a;
  int64_t runs;    // runs of TL frames
  int32_t TL, nw;  // nw: waves along the channels
  float* part;     // [B * runs][W + 1][D]
};

__device__ __forceinline__ int64_t own_of(const sed_conv_args& a, int64_t b) {
  return a.frames ? std::max<int64_t>(0, std::min<int64_t>(a.L, a.frames[b])) : a.L;
}
__device__ __forceinline__ int64_t row_of(const sed_conv_args& a, int64_t own, int64_t i) { return a.reverse && i < own ? own - 1 - i : i; }

// x at place i of the clip in the order of the walk: the state in front of it, nothing behind it.
template <class T>
__device__ __forceinline__ float x_at(const sed_conv_args& a, int64_t b, int64_t own, int64_t d, int64_t i) {
  if (i >= own) return 0.0f;
  if (i >= 0) return (float)static_cast<const T*>(a.x)[b * a.x_b + row_of(a, own, i) * a.x_t + d];
  return a.state && i + a.W - 1 >= 0 ? (float)static_cast<const T*>(a.state)[(b * (a.W - 1) + i + a.W - 1) * a.D + d] : 0.0f;
}

template <int V, int WM>
__device__ __forceinline__ void load_weights(const sed_conv_args& a, int64_t d, float (&w)[WM][V], float (&bias)[V]) {
  if (WM == 4 && a.W == 4 && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(a.weight + (d + c) * 4);
      bias[c] = a.bias ? a.bias[d + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < WM; ++k) w[k][c] = v[k % 4];
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    bias[c] = a.bias ? a.bias[d + c] : 0.0f;
#pragma unroll
    for (int k = 0; k < WM; ++k) w[k][c] = k >= WM - a.W ? a.weight[(d + c) * a.W + k - (WM - a.W)] : 0.0f;
  }
}

// acc + w x for tap m of WM, of which the first WM - W are none of the call's: what lies in front of its window, an infinity say, stays
// out (its weight of zero would make a NaN of it).  An instance for 2 taps is called with 1 or 2, for 8 with 5 to 8.
template <int WM>
__device__ __forceinline__ float tap(const sed_conv_args& a, int m, float w, float x, float acc) {
  constexpr int pads = WM == 2 ? 1 : WM == 8 ? 3 : 0;
  const float sum = fmaf(w, x, acc);
  return m < pads && m < WM - a.W ? acc : sum;
}

template <class T, int V>
using Vec = T __attribute__((ext_vector_type(V)));

// What a wave works on; d: the lane's first channel, or the last V where it has none (it stores nothing then).
struct Run {
  int64_t b, own, i0, i1, index;
  int64_t d;
  bool in;
};
template <int V>
__device__ __forceinline__ Run run_of(const ConvParams& p) {
  const sed_conv_args& a = p.a;
  Run r;
  unsigned q = blockIdx.x;
  r.d = (int64_t)(q % p.nw * 64 + threadIdx.x) * V;
  r.in = r.d < a.D;
  if (!r.in) r.d = a.D - V;
  q /= p.nw;
  r.index = q;
  r.b = q / (unsigned)p.runs;
  r.i0 = (int64_t)(q % (unsigned)p.runs) * p.TL;
  r.i1 = std::min<int64_t>(r.i0 + p.TL, a.L);
  r.own = own_of(a, r.b);
  return r;
}

// Row i of x in the order of the walk (i is the same for the wave): the state in front of the clip, zero behind it.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> row_at(const sed_conv_args& a, const Run& r, int64_t i) {
  const T* p = nullptr;
  if (i >= 0 && i < r.own) p = static_cast<const T*>(a.x) + r.b * a.x_b + row_of(a, r.own, i) * a.x_t;
  if (i < 0 && a.state && i + a.W - 1 >= 0) p = static_cast<const T*>(a.state) + (r.b * (a.W - 1) + i + a.W - 1) * a.D;
  if (!p) return Vec<T, V>{};
  return *reinterpret_cast<const Vec<T, V>*>(reinterpret_cast<const char*>(p) + (uint32_t)r.d * (uint32_t)sizeof(T));
}
// Row i >= 0 of the walk out of the rows `p` of a clip that has some, the last own one in place of those behind it: a load without a
// condition, whose value the caller leaves out there.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> row_in(const sed_conv_args& a, const Run& r, const void* p, int64_t step, int64_t i) {
  const int64_t row = row_of(a, r.own, std::min(i, r.own - 1));
  return *reinterpret_cast<const Vec<T, V>*>(static_cast<const char*>(p) + row * step * (int64_t)sizeof(T) + (uint32_t)r.d * (uint32_t)sizeof(T));
}

template <class T, int V>
__device__ __forceinline__ void put_row(const sed_conv_args& a, const Run& r, void* base, int64_t i, const float (&v)[V]) {
  T* p = static_cast<T*>(base) + (r.b * a.L + row_of(a, r.own, i)) * a.D;
  store_n<T, V, (V > 1)>(reinterpret_cast<T*>(reinterpret_cast<char*>(p) + (uint32_t)r.d * (uint32_t)sizeof(T)), r.in ? V : 0, v);
}

template <class T, int V, int WM, int ACT>
__global__ void __launch_bounds__(64) conv_forward_kernel(const ConvParams p) {
  const sed_conv_args& a = p.a;
  const Run r = run_of<V>(p);
  const T* x = static_cast<const T*>(a.x) + r.b * a.x_b;
  if (r.i0 >= r.own) {  // nothing of the clip's own: rows of zeros
    const float zero[V] = {};
    for (int64_t i = r.i0; i < r.i1; ++i) put_row<T, V>(a, r, a.y, i, zero);
    return;
  }
  float w[WM][V], bias[V], win[WM][V];
  Vec<T, V> next[WM];
#pragma unroll
  for (int k = 0; k < WM; ++k) next[k] = row_in<T, V>(a, r, x, a.x_t, r.i0 + k);
#pragma unroll
  for (int k = 1; k < WM; ++k) {  // row i lies in win[(i - i0) % WM]
    const Vec<T, V> v = row_at<T, V>(a, r, r.i0 - WM + k);
#pragma unroll
    for (int c = 0; c < V; ++c) win[k][c] = (float)v[c];
  }
  load_weights<V, WM>(a, r.d, w, bias);
  for (int64_t i = r.i0; i < r.i1; i += WM) {
    Vec<T, V> in[WM];
#pragma unroll
    for (int k = 0; k < WM; ++k) in[k] = next[k];
    if (i + WM < r.i1) {
#pragma unroll
      for (int k = 0; k < WM; ++k) next[k] = row_in<T, V>(a, r, x, a.x_t, i + WM + k);
    }
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      float y[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        win[k][c] = (float)in[k][c];
        float u = bias[c];
#pragma unroll
        for (int m = 0; m < WM; ++m) u = tap<WM>(a, m, w[m][c], win[(k + 1 + m) % WM][c], u);
        y[c] = i + k < r.own ? act<ACT>(u) : 0.0f;
      }
      if (i + k < r.i1) put_row<T, V>(a, r, a.y, i + k, y);
    }
  }
}

// Gradient of the run's rows: du_i = dy_i act'(u_i), dx_i = sum_j w[W-1-j] du_{i+j}; the W - 1 rows behind the run are formed
// again for it, and counted in the weight gradient by the run they belong to.
template <class T, int V, int WM, int ACT>
__global__ void __launch_bounds__(64) conv_backward_kernel(const ConvParams p) {
  const sed_conv_args& a = p.a;
  const Run r = run_of<V>(p);
  float w[WM][V], bias[V], win[WM][V], du[WM][V], dw[WM][V], db[V];
  Vec<T, V> nx[WM], ny[WM];
  const T *x = static_cast<const T*>(a.x) + r.b * a.x_b, *g = static_cast<const T*>(a.dy) + r.b * a.dy_b;
  const int64_t last = std::min(r.i1, r.own);  // the run's own rows end here
  if (r.i0 < last) {
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      nx[k] = row_in<T, V>(a, r, x, a.x_t, r.i0 + k);
      ny[k] = row_in<T, V>(a, r, g, a.dy_t, r.i0 + k);
    }
  }
#pragma unroll
  for (int k = 1; k < WM; ++k) {
    const Vec<T, V> v = row_at<T, V>(a, r, r.i0 - WM + k);
#pragma unroll
    for (int c = 0; c < V; ++c) win[k][c] = (float)v[c];
  }
  load_weights<V, WM>(a, r.d, w, bias);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    db[c] = 0.0f;
#pragma unroll
    for (int k = 0; k < WM; ++k) dw[k][c] = du[k][c] = 0.0f;
  }
  const float zero[V] = {};
  for (int64_t i = std::max(r.i0, r.own); i < r.i1; ++i) put_row<T, V>(a, r, a.dx, i, zero);
  for (int64_t i = r.i0; i < last + WM - 1 && r.i0 < last; i += WM) {
    Vec<T, V> in[WM], dy[WM];
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      in[k] = nx[k];
      dy[k] = ny[k];
    }
    if (i + WM < last + WM - 1) {
#pragma unroll
      for (int k = 0; k < WM; ++k) {
        nx[k] = row_in<T, V>(a, r, x, a.x_t, i + WM + k);
        ny[k] = row_in<T, V>(a, r, g, a.dy_t, i + WM + k);
      }
    }
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      const bool counts = i + k < last;
      const int64_t at = i + k - (WM - 1);
      float dx[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        win[k][c] = (float)in[k][c];
        float u = bias[c];
#pragma unroll
        for (int m = 0; m < WM; ++m) u = tap<WM>(a, m, w[m][c], win[(k + 1 + m) % WM][c], u);
        du[k][c] = i + k < r.own ? (float)dy[k][c] * act_slope<ACT>(u) : 0.0f;
      }
      if (counts) {
#pragma unroll
        for (int c = 0; c < V; ++c) {
          db[c] += du[k][c];
#pragma unroll
          for (int m = 0; m < WM; ++m) dw[m][c] = fmaf(du[k][c], win[(k + 1 + m) % WM][c], dw[m][c]);
        }
      }
      if (at >= r.i0 && at < last) {
        // row i + k - (WM - 1): du of that row and of the WM - 1 behind it
#pragma unroll
        for (int c = 0; c < V; ++c) {
          dx[c] = 0.0f;
#pragma unroll
          for (int j = 0; j < WM; ++j) dx[c] = tap<WM>(a, WM - 1 - j, w[WM - 1 - j][c], du[(k + 1 + j) % WM][c], dx[c]);
        }
        const int64_t late = at - (r.own - (a.W - 1));  // row of the state that the call returned
        if (a.dstate_out && late >= 0) {
          const T* e = static_cast<const T*>(a.dstate_out) + (r.b * (a.W - 1) + late) * a.D + r.d;
#pragma unroll
          for (int c = 0; c < V; ++c) dx[c] += (float)e[c];
        }
        put_row<T, V>(a, r, a.dx, at, dx);
      }
    }
  }
  if (!r.in) return;
  float* to = p.part + r.index * (a.W + 1) * a.D + r.d;
#pragma unroll
  for (int k = 0; k < WM; ++k)
    if (k >= WM - a.W) store_n<float, V, (V > 1)>(to + (int64_t)(k - (WM - a.W)) * a.D, V, dw[k]);
  store_n<float, V, (V > 1)>(to + (int64_t)a.W * a.D, V, db);
}

// The last W - 1 rows the clip has seen, its state in front of them where it has fewer of its own.
template <class T>
__global__ void __launch_bounds__(256) conv_state_kernel(const sed_conv_args a) {
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, n = a.W - 1;
  if (q >= a.B * n * a.D) return;
  const int64_t d = q % a.D, r = q / a.D % n, b = q / a.D / n, own = own_of(a, b);
  static_cast<T*>(a.state_out)[q] = (T)x_at<T>(a, b, own, d, own - n + r);
}

// Gradient of the state: row r is place r - (W - 1) in front of the clip.
template <class T, int ACT>
__global__ void __launch_bounds__(256) conv_state_grad_kernel(const sed_conv_args a) {
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, n = a.W - 1;
  if (q >= a.B * n * a.D) return;
  const int64_t d = q % a.D, r = q / a.D % n, b = q / a.D / n, own = own_of(a, b), i = r - n;
  float s = 0.0f;
  for (int64_t t = 0; t <= i + a.W - 1 && t < own; ++t) {
    float u = a.bias ? a.bias[d] : 0.0f;
    for (int k = 0; k < a.W; ++k) u = fmaf(a.weight[d * a.W + k], x_at<T>(a, b, own, d, t - (a.W - 1) + k), u);
    const float g = (float)static_cast<const T*>(a.dy)[b * a.dy_b + row_of(a, own, t) * a.dy_t + d] * act_slope<ACT>(u);
    s = fmaf(a.weight[d * a.W + (i - t + a.W - 1)], g, s);
  }
  const int64_t late = i - (own - n);
  if (a.dstate_out && late >= 0) s += (float)static_cast<const T*>(a.dstate_out)[(b * n + late) * a.D + d];
  static_cast<T*>(a.dstate)[q] = rounded<T>(s);
}

// dw [D][W] and db [D] out of the runs' sums [rows][W + 1][D].
__global__ void __launch_bounds__(1024) conv_param_kernel(const ConvParams p, int64_t rows, int64_t step) {
  const sed_conv_args& a = p.a;
  const int64_t cols = (int64_t)(a.W + 1) * a.D, c = (int64_t)blockIdx.x * kColumns + threadIdx.x % kColumns;
  const float t = column_sum(p.part + c, rows, step, c < cols);
  if (threadIdx.x >= kColumns || c >= cols) return;
  const int64_t k = c / a.D, d = c % a.D;
  if (k < a.W)
    a.dw[d * a.W + k] = t;
  else if (a.db)
    a.db[d] = t;
}

// One frame: the state moves up by a row in place.  A thread owns V channels of a stream.
template <class T, int V, bool VEC, int WM, int ACT>
__global__ void __launch_bounds__(256) conv_step_kernel(const sed_conv_args a, int nv) {
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= a.B * nv) return;
  const int64_t d = q % nv * V, b = q / nv;
  float w[WM][V], bias[V], win[WM][V], y[V];
  load_weights<V, WM>(a, d, w, bias);
  T* st = static_cast<T*>(a.state_out) + b * (a.W - 1) * a.D + d;
#pragma unroll
  for (int k = 0; k < WM - 1; ++k) {
    const int r = k - (WM - a.W);
    load_n<T, V, VEC>(st + (r >= 0 ? (int64_t)r * a.D : 0), r >= 0 ? V : 0, win[k]);
  }
  load_n<T, V, VEC>(static_cast<const T*>(a.x) + b * a.x_b + d, V, win[WM - 1]);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    float u = bias[c];
#pragma unroll
    for (int k = 0; k < WM; ++k) u = fmaf(w[k][c], win[k][c], u);
    y[c] = act<ACT>(u);
  }
#pragma unroll
  for (int k = 1; k < WM; ++k) {
    const int r = k - 1 - (WM - a.W);
    if (r >= 0) store_n<T, V, VEC>(st + (int64_t)r * a.D, V, win[k]);
  }
  store_n<T, V, VEC>(static_cast<T*>(a.y) + b * a.D + d, V, y);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_args(const sed_conv_args* a) {
  if (!a || a->B < 0 || a->L < 0 || a->D < 1 || a->D > (1 << 24) || a->W < 1 || a->W > 8) return SED_ERR_BAD_ARG;
  if (a->dtype != SED_F32 && a->dtype != SED_BF16 && a->dtype != SED_F16) return SED_ERR_BAD_ARG;
  if (a->act != SED_ACT_NONE && a->act != SED_ACT_SILU) return SED_ERR_BAD_ARG;
  if (a->B > 0 && a->L > 0 && (!a->x || !a->weight)) return SED_ERR_BAD_ARG;
  return SED_OK;
}

// Channels a lane takes: 4 where every row allows such loads and at least one wave of lanes is filled, else 1.
int vector_of(const sed_conv_args& a) {
  const int64_t bytes = a.dtype == SED_F32 ? 16 : 8;
  const auto ok = [&](const void* p) { return aligned(p, bytes); };
  const bool vec = a.D % 4 == 0 && a.D >= 256 && a.x_b % 4 == 0 && a.x_t % 4 == 0 && a.dy_b % 4 == 0 && a.dy_t % 4 == 0 && ok(a.x) && ok(a.dy) &&
                   ok(a.y) && ok(a.dx) && ok(a.state) && ok(a.state_out);
  return vec ? 4 : 1;
}

// Frames of a run: long runs read fewer rows twice and leave fewer sums behind; short ones make waves enough for the card
// (4096, four for each vector unit).
int run_frames(int64_t B, int64_t L, int64_t nw, bool back) {
  int TL = back ? 64 : 32;
  while (TL > 8 && B * nw * ((L + TL - 1) / TL) < 4096) TL /= 2;
  return TL;
}
int64_t waves_along(int64_t D, int V) { return (D / V + 63) / 64; }

// The gradient's lane takes 2 channels in place of 4 where more than 4 taps would leave no room for them (254 registers, one wave a
// vector unit, fp32 with 36 of them spilt).  16 x 4096 x 1536 with 8 taps: bf16 276 us with 4, 248 with 2, 312 with 1; fp32 402, 319, 324.
constexpr int back_vector(int V, int taps) { return V == 4 && taps > 4 ? 2 : V; }

template <class T, int V, int WM>
int launch_forward(const ConvParams& p, hipStream_t s) {
  const sed_conv_args& a = p.a;
  const int64_t grid = a.B * p.runs * p.nw;
  if (!grid_fits(grid, 64)) return SED_ERR_CAPACITY;
  if (a.act == SED_ACT_SILU)
    conv_forward_kernel<T, V, WM, SED_ACT_SILU><<<(unsigned)grid, 64, 0, s>>>(p);
  else
    conv_forward_kernel<T, V, WM, SED_ACT_NONE><<<(unsigned)grid, 64, 0, s>>>(p);
  return seq_status(hipGetLastError());
}

template <class T, int V, int WM>
int launch_backward(const ConvParams& p, hipStream_t s) {
  const sed_conv_args& a = p.a;
  const int64_t grid = a.B * p.runs * p.nw;
  if (!grid_fits(grid, 64)) return SED_ERR_CAPACITY;
  if (a.act == SED_ACT_SILU)
    conv_backward_kernel<T, V, WM, SED_ACT_SILU><<<(unsigned)grid, 64, 0, s>>>(p);
  else
    conv_backward_kernel<T, V, WM, SED_ACT_NONE><<<(unsigned)grid, 64, 0, s>>>(p);
  const int64_t cols = (a.W + 1) * a.D;
  int64_t rows = a.B * p.runs, step = cols;
  fold_rows(p.part, rows, step, cols, s);
  conv_param_kernel<<<(unsigned)((cols + kColumns - 1) / kColumns), 1024, 0, s>>>(p, rows, step);
  return seq_status(hipGetLastError());
}

template <class T, int V, int WM>
int launch_step(const sed_conv_args& a, hipStream_t s) {
  const int nv = (int)(a.D / V);
  const int64_t grid = (a.B * nv + 255) / 256;
  if (!grid_fits(grid, 256)) return SED_ERR_CAPACITY;
  if (a.act == SED_ACT_SILU)
    conv_step_kernel<T, V, (V > 1), WM, SED_ACT_SILU><<<(unsigned)grid, 256, 0, s>>>(a, nv);
  else
    conv_step_kernel<T, V, (V > 1), WM, SED_ACT_NONE><<<(unsigned)grid, 256, 0, s>>>(a, nv);
  return seq_status(hipGetLastError());
}

enum Kind { FORWARD, BACKWARD, STEP };

template <class T, int V, int WM>
int go_kind(const ConvParams& p, Kind kind, hipStream_t s) {
  if (kind == STEP) return launch_step<T, V, WM>(p.a, s);
  if (kind == FORWARD) return launch_forward<T, V, WM>(p, s);
  return launch_backward<T, back_vector(V, WM), WM>(p, s);
}

template <class T, int V>
int go_w(const ConvParams& p, Kind kind, hipStream_t s) {
  if (p.a.W <= 2) return go_kind<T, V, 2>(p, kind, s);
  if (p.a.W == 3) return go_kind<T, V, 3>(p, kind, s);
  if (p.a.W == 4) return go_kind<T, V, 4>(p, kind, s);
  return go_kind<T, V, 8>(p, kind, s);
}

template <class T>
int go(const ConvParams& p, Kind kind, int V, hipStream_t s) {
  const sed_conv_args& a = p.a;
  const bool state = a.W > 1 && (kind == FORWARD ? a.state_out != nullptr : kind == BACKWARD && a.dstate);
  const int64_t grid = (a.B * (a.W - 1) * a.D + 255) / 256;
  if (state && !grid_fits(grid, 256)) return SED_ERR_CAPACITY;
  const int rc = V == 4 ? go_w<T, 4>(p, kind, s) : go_w<T, 1>(p, kind, s);
  if (rc != SED_OK || !state) return rc;
  if (kind == FORWARD) {
    conv_state_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
  } else if (a.act == SED_ACT_SILU) {
    conv_state_grad_kernel<T, SED_ACT_SILU><<<(unsigned)grid, 256, 0, s>>>(a);
  } else {
    conv_state_grad_kernel<T, SED_ACT_NONE><<<(unsigned)grid, 256, 0, s>>>(a);
  }
  return seq_status(hipGetLastError());
}

int run(const sed_conv_args* args, Kind kind, void* stream) {
  ConvParams p{};
  p.a = *args;
  const int V = vector_of(p.a);
  p.nw = (int32_t)waves_along(p.a.D, kind == BACKWARD ? back_vector(V, p.a.W) : V);
  p.TL = run_frames(p.a.B, p.a.L, p.nw, kind == BACKWARD);
  p.runs = (p.a.L + p.TL - 1) / p.TL;
  if (kind == BACKWARD) {
    if (!p.a.ws || p.a.ws_bytes < 4 * p.a.B * p.runs * (p.a.W + 1) * p.a.D || !aligned(p.a.ws, 16)) return SED_ERR_CAPACITY;
    p.part = static_cast<float*>(p.a.ws);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.a.dtype == SED_F32) return go<float>(p, kind, V, s);
  if (p.a.dtype == SED_BF16) return go<bf16>(p, kind, V, s);
  return go<f16>(p, kind, V, s);
}

}  // namespace
}  // namespace sed

extern "C" int64_t sed_causal_conv_workspace(int64_t B, int64_t L, int64_t D, int32_t W) {
  if (B < 0 || L < 0 || D < 1 || W < 1 || W > 8) return SED_ERR_BAD_ARG;
  int64_t most = 0;
  for (const int V : {1, sed::back_vector(4, W)}) {
    if (D % V) continue;
    const int TL = sed::run_frames(B, L, sed::waves_along(D, V), true);
    most = std::max<int64_t>(most, 4 * B * ((L + TL - 1) / TL) * (W + 1) * D);
  }
  return most;
}

extern "C" int sed_causal_conv_forward(const sed_conv_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->y) return SED_ERR_BAD_ARG;
  return sed::run(args, sed::FORWARD, stream);
}

extern "C" int sed_causal_conv_backward(const sed_conv_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->dy || !args->dx || !args->dw || (args->dstate && !args->state)) return SED_ERR_BAD_ARG;
  return sed::run(args, sed::BACKWARD, stream);
}

extern "C" int sed_causal_conv_step(const sed_conv_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->y || (args->W > 1 && !args->state_out) || args->L != 1) return SED_ERR_BAD_ARG;
  return sed::run(args, sed::STEP, stream);
}
