// Causal depthwise convolution along the frames of a clip, with bias and SiLU, its gradient and its one-frame form, gfx950.
//
//   u_t[d] = bias[d] + sum_k w[d,k] x_{t-W+1+k}[d],  y = act(u),  x before the first frame = state (or 0)
//
// Bound: HBM (read x, write y; the gradient reads x and dy and writes dx).  A thread owns V neighbouring channels (16 bytes)
// and a run of frames, keeps the window of WM rows and the weights in registers, and meets every row once but for the
// WM - 1 rows in front of its run.  Rows are loaded WM at a time before they are used.  WM is W rounded up to 2, 4 or 8:
// the weights in front are zero.  The weight gradient is summed per thread over its run, written once per run and added
// over the runs in a fixed order.  Sums are fp32 and every output is rounded once.
#include "seq_core.h"

#include <algorithm>

namespace sed {
namespace {

struct ConvParams {
  sed_conv_args a;
  int64_t runs;  // runs of TL frames
  int32_t TL, nv;
  float* part;   // [B * runs][W + 1][D]
};

template <class T, int V, bool VEC>
struct Lane {
  int64_t d, own, b, run;
  int n;
};

__device__ __forceinline__ int64_t own_of(const sed_conv_args& a, int64_t b) {
  return a.frames ? std::max<int64_t>(0, std::min<int64_t>(a.L, a.frames[b])) : a.L;
}
__device__ __forceinline__ int64_t row_of(const sed_conv_args& a, int64_t own, int64_t i) { return a.reverse && i < own ? own - 1 - i : i; }

// x at place i of the clip in the order of the walk: the state in front of it, nothing behind it.
template <class T, int V, bool VEC>
__device__ __forceinline__ void x_at(const sed_conv_args& a, int64_t b, int64_t own, int64_t d, int64_t i, float (&v)[V]) {
  const T* p = static_cast<const T*>(a.x) + b * a.x_b + d;
  int n = V;
  if (i >= 0) {
    n = i < own ? V : 0;
    p += (n ? row_of(a, own, i) : 0) * a.x_t;
  } else {
    n = a.state && i + a.W - 1 >= 0 ? V : 0;
    if (n) p = static_cast<const T*>(a.state) + (b * (a.W - 1) + i + a.W - 1) * a.D + d;
  }
  load_n<T, V, VEC>(p, n, v);
}

template <int V, int WM>
__device__ __forceinline__ void load_weights(const sed_conv_args& a, int64_t d, float (&w)[WM][V], float (&bias)[V]) {
#pragma unroll
  for (int c = 0; c < V; ++c) {
    bias[c] = a.bias ? a.bias[d + c] : 0.0f;
#pragma unroll
    for (int k = 0; k < WM; ++k) w[k][c] = k >= WM - a.W ? a.weight[(d + c) * a.W + k - (WM - a.W)] : 0.0f;
  }
}

template <class T, int V, bool VEC, int WM, int ACT>
__global__ void __launch_bounds__(256) conv_forward_kernel(const ConvParams p) {
  const sed_conv_args& a = p.a;
  int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= a.B * p.runs * p.nv) return;
  const int64_t d = q % p.nv * V;
  q /= p.nv;
  const int64_t i0 = q % p.runs * p.TL, b = q / p.runs, own = own_of(a, b), i1 = std::min<int64_t>(i0 + p.TL, a.L);
  float w[WM][V], bias[V], win[WM][V];
  load_weights<V, WM>(a, d, w, bias);
#pragma unroll
  for (int k = 1; k < WM; ++k) x_at<T, V, VEC>(a, b, own, d, i0 - WM + k, win[k]);  // row i lies in win[(i - i0) % WM]
  for (int64_t i = i0; i < i1; i += WM) {
    float in[WM][V];
#pragma unroll
    for (int k = 0; k < WM; ++k) x_at<T, V, VEC>(a, b, own, d, i + k, in[k]);
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      float y[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        win[k][c] = in[k][c];
        float u = bias[c];
#pragma unroll
        for (int m = 0; m < WM; ++m) u = fmaf(w[m][c], win[(k + 1 + m) % WM][c], u);
        y[c] = i + k < own ? act<ACT>(u) : 0.0f;
      }
      if (i + k < i1) store_n<T, V, VEC>(static_cast<T*>(a.y) + (b * a.L + row_of(a, own, i + k)) * a.D + d, V, y);
    }
  }
}

// Gradient of the run's rows: du_i = dy_i act'(u_i), dx_i = sum_j w[W-1-j] du_{i+j}; the W - 1 rows behind the run are formed
// again for it, and counted in the weight gradient by the run they belong to.
template <class T, int V, bool VEC, int WM, int ACT>
__global__ void __launch_bounds__(256) conv_backward_kernel(const ConvParams p) {
  const sed_conv_args& a = p.a;
  int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= a.B * p.runs * p.nv) return;
  const int64_t d = q % p.nv * V;
  q /= p.nv;
  const int64_t run = q, i0 = q % p.runs * p.TL, b = q / p.runs, own = own_of(a, b), i1 = std::min<int64_t>(i0 + p.TL, a.L);
  float w[WM][V], bias[V], win[WM][V], du[WM][V], dw[WM][V], db[V];
  load_weights<V, WM>(a, d, w, bias);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    db[c] = 0.0f;
#pragma unroll
    for (int k = 0; k < WM; ++k) dw[k][c] = du[k][c] = 0.0f;
  }
#pragma unroll
  for (int k = 1; k < WM; ++k) x_at<T, V, VEC>(a, b, own, d, i0 - WM + k, win[k]);
  for (int64_t i = i0; i < i1 + WM - 1; i += WM) {
    float in[WM][V], dy[WM][V];
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      x_at<T, V, VEC>(a, b, own, d, i + k, in[k]);
      const bool mine = i + k < own;
      load_n<T, V, VEC>(static_cast<const T*>(a.dy) + b * a.dy_b + (mine ? row_of(a, own, i + k) : 0) * a.dy_t + d, mine ? V : 0, dy[k]);
    }
#pragma unroll
    for (int k = 0; k < WM; ++k) {
      const bool counts = i + k < i1;  // rows behind the clip's own have dy = 0
      float dx[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        win[k][c] = in[k][c];
        float u = bias[c];
#pragma unroll
        for (int m = 0; m < WM; ++m) u = fmaf(w[m][c], win[(k + 1 + m) % WM][c], u);
        const float g = i + k < own ? dy[k][c] * act_slope<ACT>(u) : 0.0f;
        du[k][c] = g;
        const float gc = counts ? g : 0.0f;
        db[c] += gc;
#pragma unroll
        for (int m = 0; m < WM; ++m) dw[m][c] = fmaf(gc, win[(k + 1 + m) % WM][c], dw[m][c]);
        // row i + k - (WM - 1): du of that row and the WM - 1 behind it
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < WM; ++j) s = fmaf(w[WM - 1 - j][c], du[(k + 1 + j) % WM][c], s);
        dx[c] = s;
      }
      const int64_t r = i + k - (WM - 1);
      if (r >= i0 && r < i1) {
        const int64_t late = r - (own - (a.W - 1));  // row of the state that the call returned
        if (r >= own) {
#pragma unroll
          for (int c = 0; c < V; ++c) dx[c] = 0.0f;
        } else if (a.dstate_out && late >= 0) {
          float e[V];
          load_n<T, V, VEC>(static_cast<const T*>(a.dstate_out) + (b * (a.W - 1) + late) * a.D + d, V, e);
#pragma unroll
          for (int c = 0; c < V; ++c) dx[c] += e[c];
        }
        store_n<T, V, VEC>(static_cast<T*>(a.dx) + (b * a.L + row_of(a, own, r)) * a.D + d, V, dx);
      }
    }
  }
  float* to = p.part + run * (a.W + 1) * a.D + d;
#pragma unroll
  for (int k = 0; k < WM; ++k)
    if (k >= WM - a.W) {
#pragma unroll
      for (int c = 0; c < V; ++c) to[(int64_t)(k - (WM - a.W)) * a.D + c] = dw[k][c];
    }
#pragma unroll
  for (int c = 0; c < V; ++c) to[(int64_t)a.W * a.D + c] = db[c];
}

// The last W - 1 rows the clip has seen, its state in front of them where it has fewer of its own.
template <class T>
__global__ void __launch_bounds__(256) conv_state_kernel(const sed_conv_args a) {
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, n = a.W - 1;
  if (q >= a.B * n * a.D) return;
  const int64_t d = q % a.D, r = q / a.D % n, b = q / a.D / n, own = own_of(a, b);
  float v[1];
  x_at<T, 1, false>(a, b, own, d, own - n + r, v);
  static_cast<T*>(a.state_out)[q] = (T)v[0];
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
    for (int k = 0; k < a.W; ++k) {
      float v[1];
      x_at<T, 1, false>(a, b, own, d, t - (a.W - 1) + k, v);
      u = fmaf(a.weight[d * a.W + k], v[0], u);
    }
    const float g = (float)static_cast<const T*>(a.dy)[b * a.dy_b + row_of(a, own, t) * a.dy_t + d] * act_slope<ACT>(u);
    s = fmaf(a.weight[d * a.W + (i - t + a.W - 1)], g, s);
  }
  const int64_t late = i - (own - n);
  if (a.dstate_out && late >= 0) s += (float)static_cast<const T*>(a.dstate_out)[(b * n + late) * a.D + d];
  static_cast<T*>(a.dstate)[q] = (T)s;
}

// dw [D][W] and db [D] out of the runs' sums [rows][W + 1][D], a thread for every 4th row, added in order.
__global__ void __launch_bounds__(1024) conv_param_kernel(const ConvParams p) {
  const sed_conv_args& a = p.a;
  __shared__ float s[16][64];
  const int64_t cols = (int64_t)(a.W + 1) * a.D, c = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
  const int ty = threadIdx.x / 64;
  const int64_t rows = a.B * p.runs;
  float v[4] = {0, 0, 0, 0};
  if (c < cols) {
    int64_t r = ty;
    for (; r + 48 < rows; r += 64)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += p.part[(r + 16 * k) * cols + c];
    for (; r < rows; r += 16) v[0] += p.part[r * cols + c];
  }
  s[ty][threadIdx.x % 64] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (ty == 0 && c < cols) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += s[k][threadIdx.x];
    const int64_t k = c / a.D, d = c % a.D;
    if (k < a.W)
      a.dw[d * a.W + k] = t;
    else if (a.db)
      a.db[d] = t;
  }
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
  if (!a || a->B < 0 || a->L < 0 || a->D < 1 || a->W < 1 || a->W > 8) return SED_ERR_BAD_ARG;
  if (a->dtype != SED_F32 && a->dtype != SED_BF16 && a->dtype != SED_F16) return SED_ERR_BAD_ARG;
  if (a->act != SED_ACT_NONE && a->act != SED_ACT_SILU) return SED_ERR_BAD_ARG;
  if (a->B > 0 && a->L > 0 && (!a->x || !a->weight)) return SED_ERR_BAD_ARG;
  return SED_OK;
}

int vector_of(const sed_conv_args& a) {
  const int V = a.dtype == SED_F32 ? 4 : 8;
  const auto ok = [&](const void* p) { return aligned(p, 16); };
  const bool vec = a.D % V == 0 && a.x_b % V == 0 && a.x_t % V == 0 && (!a.dy || (a.dy_b % V == 0 && a.dy_t % V == 0)) && ok(a.x) && ok(a.dy) &&
                   ok(a.y) && ok(a.dx) && ok(a.state) && ok(a.state_out) && ok(a.dstate_out);
  return vec ? V : 1;
}

// Frames of a run: long runs read fewer rows twice and leave fewer sums behind; short ones keep 256 compute units busy
// (64 Ki threads at least).
int run_frames(int64_t B, int64_t L, int64_t nv, bool back) {
  int TL = back ? 64 : 16;
  while (TL > 8 && B * nv * ((L + TL - 1) / TL) < 65536) TL /= 2;
  return TL;
}

template <class T, int V, bool VEC, int WM>
int launch(const ConvParams& p, bool back, hipStream_t s) {
  const sed_conv_args& a = p.a;
  const int64_t grid = (a.B * p.runs * p.nv + 255) / 256;
  if (grid > 0x7fffffff) return SED_ERR_CAPACITY;
  const unsigned n = (unsigned)grid;
  if (!back) {
    if (a.act == SED_ACT_SILU)
      conv_forward_kernel<T, V, VEC, WM, SED_ACT_SILU><<<n, 256, 0, s>>>(p);
    else
      conv_forward_kernel<T, V, VEC, WM, SED_ACT_NONE><<<n, 256, 0, s>>>(p);
    return seq_status(hipGetLastError());
  }
  if (a.act == SED_ACT_SILU)
    conv_backward_kernel<T, V, VEC, WM, SED_ACT_SILU><<<n, 256, 0, s>>>(p);
  else
    conv_backward_kernel<T, V, VEC, WM, SED_ACT_NONE><<<n, 256, 0, s>>>(p);
  conv_param_kernel<<<(unsigned)(((a.W + 1) * a.D + 63) / 64), 1024, 0, s>>>(p);
  return seq_status(hipGetLastError());
}

template <class T, int V, bool VEC, int WM>
int launch_step(const sed_conv_args& a, hipStream_t s) {
  const int nv = (int)(a.D / V);
  const int64_t grid = (a.B * nv + 255) / 256;
  if (grid > 0x7fffffff) return SED_ERR_CAPACITY;
  if (a.act == SED_ACT_SILU)
    conv_step_kernel<T, V, VEC, WM, SED_ACT_SILU><<<(unsigned)grid, 256, 0, s>>>(a, nv);
  else
    conv_step_kernel<T, V, VEC, WM, SED_ACT_NONE><<<(unsigned)grid, 256, 0, s>>>(a, nv);
  return seq_status(hipGetLastError());
}

enum Kind { FORWARD, BACKWARD, STEP };

template <class T, int V, bool VEC>
int go_w(const ConvParams& p, Kind kind, hipStream_t s) {
  if (p.a.W <= 2) return kind == STEP ? launch_step<T, V, VEC, 2>(p.a, s) : launch<T, V, VEC, 2>(p, kind == BACKWARD, s);
  if (p.a.W <= 4) return kind == STEP ? launch_step<T, V, VEC, 4>(p.a, s) : launch<T, V, VEC, 4>(p, kind == BACKWARD, s);
  return kind == STEP ? launch_step<T, V, VEC, 8>(p.a, s) : launch<T, V, VEC, 8>(p, kind == BACKWARD, s);
}

template <class T, int V>
int go(const ConvParams& p, Kind kind, bool vec, hipStream_t s) {
  const sed_conv_args& a = p.a;
  int rc = vec ? go_w<T, V, true>(p, kind, s) : go_w<T, 1, false>(p, kind, s);
  if (rc != SED_OK || kind == STEP || a.W == 1) return rc;
  const int64_t grid = (a.B * (a.W - 1) * a.D + 255) / 256;
  if (grid > 0x7fffffff) return SED_ERR_CAPACITY;
  if (kind == FORWARD && a.state_out) conv_state_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
  if (kind == BACKWARD && a.dstate) {
    if (a.act == SED_ACT_SILU)
      conv_state_grad_kernel<T, SED_ACT_SILU><<<(unsigned)grid, 256, 0, s>>>(a);
    else
      conv_state_grad_kernel<T, SED_ACT_NONE><<<(unsigned)grid, 256, 0, s>>>(a);
  }
  return seq_status(hipGetLastError());
}

int run(const sed_conv_args* args, Kind kind, void* stream) {
  ConvParams p{};
  p.a = *args;
  const int V = vector_of(p.a);
  p.nv = (int32_t)(p.a.D / V);
  p.TL = run_frames(p.a.B, p.a.L, p.nv, kind == BACKWARD);
  p.runs = (p.a.L + p.TL - 1) / p.TL;
  if (kind == BACKWARD) {
    if (!p.a.ws || p.a.ws_bytes < 4 * p.a.B * p.runs * (p.a.W + 1) * p.a.D || !aligned(p.a.ws, 16)) return SED_ERR_CAPACITY;
    p.part = static_cast<float*>(p.a.ws);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.a.dtype == SED_F32) return go<float, 4>(p, kind, V > 1, s);
  if (p.a.dtype == SED_BF16) return go<bf16, 8>(p, kind, V > 1, s);
  return go<f16, 8>(p, kind, V > 1, s);
}

}  // namespace
}  // namespace sed

extern "C" int64_t sed_causal_conv_workspace(int64_t B, int64_t L, int64_t D, int32_t W) {
  if (B < 0 || L < 0 || D < 1 || W < 1 || W > 8) return SED_ERR_BAD_ARG;
  int64_t most = 0;
  for (const int V : {1, 4, 8}) {
    if (D % V) continue;
    const int TL = sed::run_frames(B, L, D / V, true);
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
