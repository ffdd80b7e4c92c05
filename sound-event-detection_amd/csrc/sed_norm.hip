// Group norm with an activation on channels-last maps (B, T, F, C), over a clip's own frames, and its gradient, for gfx950.
//
//   y = act((x - mean[b,g]) rstd[b,g] w[c] + bias[c]),  mean and variance over the clip's frames x F x the group's channels
//
// Bound: HBM.  The maps are walked row by row (a row = the C channels of one place), 16 bytes a lane, lanes along channels, so
// every access is whole lines whatever the group's width.  Every lane sums its own channels relative to the first value it
// meets there (a far mean costs no precision), joined per channel, then per group with the exact formula for joined means.
// The gradient needs two sums a group, sum q and sum q n (q = du w, n the normalised value), which follow from the channels'
// sums of du and du n: those are the bias' and the weight's gradients at the same time.
// Two walks over a map are what a grid without a barrier can do: the second one goes backwards, so that what the memory-side
// cache still holds is read from there.  Groups small enough for one workgroup's registers are read once, in one launch.
//
// Measured (MI355X): 32 x 1001 x 64 x 64 bf16 SiLU (262 MB a map): statistics 59 us (4.4 TB/s), output 93 us (5.6 TB/s), the
// gradient's sums 115 us (4.6 TB/s), the gradient 136 us (5.8 TB/s); a 1 GiB copy reaches 5.1.  Four walks of 8 clips each were no
// faster than one of 32.  64 x 862 x 768 GELU with lengths of their own: 37 us for the output (vector unit: 24 slots a value).
#include "seq_core.h"

#include <algorithm>

namespace sed {
namespace {

struct NormParams {
  sed_norm_args a;
  int64_t S;         // places of a clip
  int32_t nv, nb;    // vectors of a row, lanes along a row
  int32_t half;      // half the lanes of a channel, rounded up to a power of two
  int32_t blocks;    // blocks a clip is cut into
  int32_t late;      // the same for the second walk
  float* part;       // [B][blocks][2][C]: (mean, sum of squares about it), or (sum du, sum du n)
  float* chan;       // [B][2][C]
  float* gsum;       // [B][G][2]: means of q and q n
};

__device__ __forceinline__ int64_t own_of(const NormParams& p, int64_t b) {
  const sed_norm_args& a = p.a;
  const int64_t t = a.frames ? std::max<int64_t>(0, std::min<int64_t>(a.T, a.frames[b])) : a.T;
  return t * a.F;
}

// First of a clip's n places that block k of `blocks` takes: even parts, so that clips of other lengths keep every block (and
// every compute unit) as busy; parts of fixed length would leave the same units without work in clip after clip.
__device__ __forceinline__ int64_t part_begin(int blocks, int64_t n, int64_t k) {
  return n < (1 << 18) ? (int64_t)((uint32_t)n * (uint32_t)k / (uint32_t)blocks) : n * k / blocks;  // blocks <= 8192
}

struct Cell {
  int64_t b, block, r0, r1, z0, z1, c;  // the clip's own places of the block, and the ones behind that it clears
  int ty, step;
  bool in;
};
// LATE: the second walk over the map goes from its end, which the first one read last and the memory-side cache still holds.
template <int V, bool LATE>
__device__ __forceinline__ Cell cell(const NormParams& p) {
  Cell q;
  q.b = LATE ? p.a.B - 1 - blockIdx.y : blockIdx.y;
  const int blocks = LATE ? p.late : p.blocks;
  q.block = LATE ? blocks - 1 - blockIdx.x : blockIdx.x;
  const int64_t own = own_of(p, q.b);
  q.r0 = part_begin(blocks, own, q.block);
  q.r1 = part_begin(blocks, own, q.block + 1);
  q.z0 = own + part_begin(blocks, p.S - own, q.block);
  q.z1 = own + part_begin(blocks, p.S - own, q.block + 1);
  const int tx = threadIdx.x % p.nb, v = blockIdx.z * p.nb + tx;
  q.ty = threadIdx.x / p.nb;
  q.step = 256 / p.nb;
  q.c = (int64_t)v * V;
  q.in = v < p.nv && q.ty < q.step;
  return q;
}

// Sums of a block per channel: the lanes of a channel put (count, value, value) into LDS, lane 0 of it joins them.
template <class T, int V, bool VEC>
__global__ void __launch_bounds__(256) norm_stats_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  const Cell q = cell<V, false>(p);
  const int64_t end = q.r1;
  if (q.r0 >= end) return;
  __shared__ float s_m[256][V + 1], s_v[256][V + 1];
  __shared__ int s_n[256];
  float k[V], s1[V], s2[V];
  int n = 0;
  if (q.in) {
    const T* x = static_cast<const T*>(a.x) + q.b * p.S * a.C + q.c;
    int64_t r = q.r0 + q.ty;
    if (r < end) {
      float m2[V];
      load_n<T, V, VEC>(x + r * a.C, V, k);
#pragma unroll
      for (int c = 0; c < V; ++c) s1[c] = s2[c] = 0.0f;
      n = 1;
      r += q.step;
      const auto walk = [&](int64_t stop) {
        int more = 0;
#pragma unroll 4
        for (; r < stop; r += q.step) {
          float v[V];
          load_n<T, V, VEC>(x + r * a.C, V, v);
          ++more;
#pragma unroll
          for (int c = 0; c < V; ++c) {
            const float e = v[c] - k[c];
            s1[c] += e;
            s2[c] = fmaf(e, e, s2[c]);
          }
        }
        return more;
      };
      n += walk(std::min(end, r + 15 * q.step));
      const float inv = 1.0f / (float)n;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float m = s1[c] * inv;
        k[c] += m;
        m2[c] = fmaf(-m, s1[c], s2[c]);
      }
      // The first value may lie far from the others (a recording that begins with a click): after 16, 128, 1024 .. rows the next are
      // summed relative to the mean of those, which is no further off than a fraction of what the sum of squares holds.
      while (r < end) {
#pragma unroll
        for (int c = 0; c < V; ++c) s1[c] = s2[c] = 0.0f;
        const int more = walk(std::min(end, r + (int64_t)(7 * n) * q.step));
        const float inv = 1.0f / (float)more, all = 1.0f / (float)(n + more), part = (float)n * all;
        n += more;
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float d = s1[c] * inv;
          m2[c] += fmaf(d * s1[c], part, fmaf(-d, s1[c], s2[c]));
          k[c] = fmaf(s1[c], all, k[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < V; ++c) {
        s_m[threadIdx.x][c] = k[c];
        s_v[threadIdx.x][c] = m2[c];
      }
    }
  }
  s_n[threadIdx.x] = n;
  // the lanes of a channel in pairs, half as many each time
  for (int half = p.half; half >= 1; half /= 2) {
    __syncthreads();
    const int from = threadIdx.x + half * p.nb;
    if (q.in && q.ty < half && q.ty + half < q.step && s_n[from] > 0) {
      const float m = (float)s_n[from], mine = (float)s_n[threadIdx.x], part = m / (mine + m);
      s_n[threadIdx.x] += s_n[from];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float e = s_m[from][c] - s_m[threadIdx.x][c];
        s_m[threadIdx.x][c] = fmaf(e, part, s_m[threadIdx.x][c]);
        s_v[threadIdx.x][c] += fmaf(e * e, mine * part, s_v[from][c]);
      }
    }
  }
  if (q.in && q.ty == 0) {
    float* to = p.part + (q.b * p.blocks + q.block) * 2 * a.C + q.c;
    float mean[V], var[V];
#pragma unroll
    for (int c = 0; c < V; ++c) mean[c] = s_m[threadIdx.x][c], var[c] = s_v[threadIdx.x][c];
    store_n<float, V, false>(to, V, mean);
    store_n<float, V, false>(to + a.C, V, var);
  }
}

__device__ __forceinline__ float block_sum(float v, float* s) {
  v = wave_sum(v);
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

constexpr int kBlocks = 2048;  // of a clip at most, in the walk that leaves sums

// Joins the blocks of a clip per channel, 16 channels a workgroup and a thread for every 64th block, all of which it holds: into the
// first block's place, or the gradient's sums into `chan`.  For clips of more blocks and channels a group than one workgroup
// joins in passing (1 x 1001 x 64 x 256 in one group: 1936 us by norm_join_kernel alone).
template <bool BACK>
__global__ void __launch_bounds__(1024) norm_channel_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  constexpr int W = 16, H = 1024 / W, HELD = kBlocks / H;
  __shared__ float s_1[H][W + 1], s_2[H][W + 1];
  const int lane = threadIdx.x % W, row = threadIdx.x / W;
  const int64_t b = blockIdx.y, at = (int64_t)blockIdx.x * W + lane, c = std::min(at, a.C - 1), own = own_of(p, b);
  float* part = p.part + b * p.blocks * 2 * a.C + c;
  // sums over the rows, in pairs
  const auto all = [&](float (&s)[H][W + 1], float v) {
    s[row][lane] = v;
    for (int half = H / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (row < half) s[row][lane] += s[row + half][lane];
    }
    __syncthreads();
    return s[0][lane];
  };
  float m[HELD], v[HELD], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int k = row + h * H;
    m[h] = v[h] = 0.0f;
    if (k < p.blocks) {
      m[h] = part[(int64_t)k * 2 * a.C];
      v[h] = part[(int64_t)k * 2 * a.C + a.C];
    }
  }
  if constexpr (BACK) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      s1 += m[h];
      s2 += v[h];
    }
    s1 = all(s_1, s1);
    s2 = all(s_2, s2);
    if (row == 0 && at < a.C) {
      p.chan[b * 2 * a.C + c] = s1;
      p.chan[b * 2 * a.C + a.C + c] = s2;
    }
  } else {
    if (own <= 0) return;
    const float first = part[(int64_t)(p.blocks - 1) * 2 * a.C];  // the last block always has places
    float n[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int k = row + h * H;
      n[h] = k < p.blocks ? (float)(part_begin(p.blocks, own, k + 1) - part_begin(p.blocks, own, k)) : 0.0f;
      if (n[h] > 0.0f) s1 = fmaf(n[h], m[h] - first, s1);  // a block without places has written nothing
    }
    const float mean = first + all(s_1, s1) / (float)own;
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (n[h] > 0.0f) s2 += fmaf(n[h] * (m[h] - mean), m[h] - mean, v[h]);
    s2 = all(s_2, s2);
    if (row == 0 && at < a.C) {
      part[0] = mean;
      part[a.C] = s2;
    }
  }
}

// mean and rstd of a (clip, group) out of the blocks' channels: the mean first, then the squares about it, so that neither a far
// mean nor an odd block costs digits.  HELD: each thread has at most HELD entries and keeps them; 0: they are read twice.  JOINED: the
// blocks are joined already.
template <int HELD, bool JOINED>
__global__ void __launch_bounds__(256) norm_join_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  __shared__ float s[4];
  const int g = blockIdx.x % (int)a.G, b = blockIdx.x / (int)a.G, cg = (int)(a.C / a.G);
  const int64_t own = own_of(p, b);
  const int n = JOINED ? cg : p.blocks * cg;  // entries
  const float total = (float)own * (float)cg;
  const float* part = p.part + (int64_t)b * p.blocks * 2 * a.C + g * cg;
  float mean = 0.0f, var = 0.0f;
  if (own > 0) {
    const auto entry = [&](int i, float& count, float& m, float& v) {
      const int q = JOINED ? 0 : i / cg;
      const float* at = part + (int64_t)q * 2 * a.C + (i - q * cg);
      count = JOINED ? (float)own : (float)(part_begin(p.blocks, own, q + 1) - part_begin(p.blocks, own, q));
      m = count > 0.0f ? at[0] : 0.0f;  // a block without places has written nothing
      v = count > 0.0f ? at[a.C] : 0.0f;
    };
    const float k = part[JOINED ? 0 : (int64_t)(p.blocks - 1) * 2 * a.C];  // means relative to one of them (the last block always has places)
    float w = 0.0f, count[HELD ? HELD : 1], m[HELD ? HELD : 1], v[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        count[h] = m[h] = v[h] = 0.0f;
        if ((int)threadIdx.x + 256 * h < n) entry(threadIdx.x + 256 * h, count[h], m[h], v[h]);
      }
#pragma unroll
      for (int h = 0; h < HELD; ++h) w = fmaf(count[h], m[h] - k, w);
    } else {
      for (int i = threadIdx.x; i < n; i += 256) {
        entry(i, count[0], m[0], v[0]);
        w = fmaf(count[0], m[0] - k, w);
      }
    }
    mean = k + block_sum(w, s) / total;
    w = 0.0f;
    if constexpr (HELD > 0) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) w += fmaf(count[h] * (m[h] - mean), m[h] - mean, v[h]);
    } else {
      for (int i = threadIdx.x; i < n; i += 256) {
        entry(i, count[0], m[0], v[0]);
        w += fmaf(count[0] * (m[0] - mean), m[0] - mean, v[0]);
      }
    }
    var = block_sum(w, s) / total;
  }
  if (threadIdx.x == 0) {
    a.mean[(int64_t)b * a.G + g] = mean;
    a.rstd[(int64_t)b * a.G + g] = 1.0f / sqrtf(var + a.eps);
  }
}

// Rows of both maps that a gradient's lane has on the way at once.  Two where a row takes the most registers (gelu, 8 channels): there
// four leave three waves a vector unit and are 1.5 % slower (32 x 1001 x 64 x 64 bf16, forward and gradient).  Four elsewhere: fp32
// gelu 869 us against 896 with two, bf16 SiLU 435 against 442 with the compiler's own order.
template <int ACT>
constexpr int grad_rows(int channels) { return ACT == SED_ACT_GELU && channels == 8 ? 2 : 4; }

// Walks rows [r, end) in steps, ROWS of them loaded from both maps before the first is worked on (then one after another: worked
// on together they would take more registers than keep four waves a vector unit).
template <class T, int V, int ROWS, class F>
__device__ __forceinline__ void walk_two(const T* x, const T* y, int64_t r, int64_t end, int step, int64_t C, F f) {
  typedef T vt __attribute__((ext_vector_type(V)));
  const auto one = [&](const vt& a, const vt& b, int64_t at) {
    float u[V], v[V];
#pragma unroll
    for (int c = 0; c < V; ++c) u[c] = (float)a[c], v[c] = (float)b[c];
    f(u, v, at);
  };
  for (; r + (ROWS - 1) * step < end; r += ROWS * step) {
    vt a[ROWS], b[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      a[k] = *reinterpret_cast<const vt*>(x + (r + k * step) * C);
      b[k] = *reinterpret_cast<const vt*>(y + (r + k * step) * C);
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      __builtin_amdgcn_sched_barrier(0);
      one(a[k], b[k], r + k * step);
    }
  }
  for (; r < end; r += step) one(*reinterpret_cast<const vt*>(x + r * C), *reinterpret_cast<const vt*>(y + r * C), r);
}

// Calls f(channel of the lane, its group) for the lane's V channels in order.
template <int V, class F>
__device__ __forceinline__ void each_group(const NormParams& p, const Cell& q, F f) {
  const int cg = (int)(p.a.C / p.a.G);
  int g = (int)q.c / cg, left = cg - ((int)q.c - g * cg);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    f(c, q.b * p.a.G + g);
    if (--left == 0) ++g, left = cg;
  }
}

// mean, scale and shift of a lane's channels: n = (x - mean) rstd, u = n w + bias.
template <int V>
__device__ __forceinline__ void channels(const NormParams& p, const Cell& q, float (&mean)[V], float (&rstd)[V], float (&w)[V], float (&bias)[V]) {
  const sed_norm_args& a = p.a;
  each_group<V>(p, q, [&](int c, int64_t g) {
    mean[c] = a.mean[g];
    rstd[c] = a.rstd[g];
    w[c] = a.weight ? a.weight[q.c + c] : 1.0f;
    bias[c] = a.bias ? a.bias[q.c + c] : 0.0f;
  });
}

template <class T, int V, bool VEC, int ACT>
__global__ void __launch_bounds__(256) norm_apply_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  const Cell q = cell<V, true>(p);
  if (!q.in) return;
  float mean[V], rstd[V], w[V], bias[V];
  channels<V>(p, q, mean, rstd, w, bias);
#pragma unroll
  for (int c = 0; c < V; ++c) w[c] *= rstd[c];
  const int64_t at = q.b * p.S * a.C + q.c;
  const T* x = static_cast<const T*>(a.x) + at;
  T* y = static_cast<T*>(a.y) + at;
#pragma unroll 4
  for (int64_t r = q.r0 + q.ty; r < q.r1; r += q.step) {
    float v[V];
    load_n<T, V, VEC>(x + r * a.C, V, v);
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = act<ACT>(fmaf(v[c] - mean[c], w[c], bias[c]));
    store_n<T, V, VEC>(y + r * a.C, V, v);
  }
  const float zero[V] = {};
  for (int64_t r = q.z0 + q.ty; r < q.z1; r += q.step) store_n<T, V, VEC>(y + r * a.C, V, zero);
}

// A (clip, group) whose values fit into a workgroup's registers: read once, its statistics taken there, written.  Lanes along the
// group's channels, V of them each, then along the places; the sums are relative to the group's first value, the squares to the
// mean that they give, and what that mean is off by is put right in both.  Groups of a clip lie side by side in memory: workgroups
// are counted so that an XCD has whole clips and its L2 the lines that two groups share.  Bound by latency or, in large batches, by
// HBM: 1 x 101 x 64 x 32 fp32 11 us (three launches of the walks: 13), 512 x 100 x 256 bf16 18 us (41), 2000 x 200 x 256 bf16 in 8
// groups 99 us for 410 MB, 4.1 TB/s (145).
template <class T, int V, int HELD, int ACT>
__global__ void __launch_bounds__(1024) norm_whole_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  typedef T vt __attribute__((ext_vector_type(V)));
  __shared__ float s[2][16];
  const unsigned item = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  if (item >= a.B * a.G) return;
  const int b = item / (unsigned)a.G, g = item % (unsigned)a.G, cg = (int)(a.C / a.G);
  const int nv = cg / V, tx = threadIdx.x % nv, ty = threadIdx.x / nv, step = blockDim.x / nv, waves = (blockDim.x + 63) / 64;
  const int own = (int)own_of(p, b), mine = ty < step ? own : 0;  // places; of this lane
  const int64_t c = g * cg + tx * V, at = b * p.S * a.C + c;
  const T* x = static_cast<const T*>(a.x) + at;
  T* y = static_cast<T*>(a.y) + at;
  vt v[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int r = ty + h * step;
    if (r < mine) v[h] = *reinterpret_cast<const vt*>(x + r * a.C);
  }
  float w[V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = a.weight ? a.weight[c + i] : 1.0f;
    bias[i] = a.bias ? a.bias[c + i] : 0.0f;
  }
  const auto all = [&](float t, float* to) {
    t = wave_sum(t);
    if (threadIdx.x % 64 == 0) to[threadIdx.x / 64] = t;
    __syncthreads();
    t = 0.0f;
    for (int i = 0; i < waves; ++i) t += to[i];
    return t;
  };
  const float k = own > 0 ? (float)static_cast<const T*>(a.x)[b * p.S * a.C + g * cg] : 0.0f;
  const float inv = own > 0 ? 1.0f / ((float)own * (float)cg) : 0.0f;
  float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int h = 0; h < HELD; ++h)
    if (ty + h * step < mine)
#pragma unroll
      for (int i = 0; i < V; ++i) s1 += (float)v[h][i] - k;
  float mean = fmaf(all(s1, s[0]), inv, k);
  s1 = 0.0f;
#pragma unroll
  for (int h = 0; h < HELD; ++h)
    if (ty + h * step < mine)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = (float)v[h][i] - mean;
        s1 += e;
        s2 = fmaf(e, e, s2);
      }
  __syncthreads();
  const float off = all(s1, s[0]) * inv, var = fmaf(all(s2, s[1]), inv, -off * off);
  mean += off;
  const float rstd = 1.0f / sqrtf(std::max(var, 0.0f) + a.eps);
  if (threadIdx.x == 0) {
    a.mean[item] = mean;
    a.rstd[item] = rstd;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] *= rstd;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int r = ty + h * step;
    if (r < mine) {
      float u[V];
#pragma unroll
      for (int i = 0; i < V; ++i) u[i] = act<ACT>(fmaf((float)v[h][i] - mean, w[i], bias[i]));
      store_n<T, V, true>(y + r * a.C, V, u);
    }
  }
  const float zero[V] = {};
  if (ty < step)
    for (int64_t r = own + ty; r < p.S; r += step) store_n<T, V, true>(y + r * a.C, V, zero);
}

template <class T, int V, bool VEC, int ACT>
__global__ void __launch_bounds__(256) norm_grad_sums_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  const Cell q = cell<V, false>(p);
  const int64_t end = q.r1;
  __shared__ float s_1[256][V + 1], s_2[256][V + 1];
  float s1[V], s2[V];
#pragma unroll
  for (int c = 0; c < V; ++c) s1[c] = s2[c] = 0.0f;
  if (q.in) {
    float mean[V], rstd[V], w[V], bias[V];
    channels<V>(p, q, mean, rstd, w, bias);
    const int64_t at = q.b * p.S * a.C + q.c;
    const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at;
    walk_two<T, V, grad_rows<ACT>(V)>(x, dy, q.r0 + q.ty, end, q.step, a.C, [&](const float(&v)[V], const float(&g)[V], int64_t) {
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float n = (v[c] - mean[c]) * rstd[c], du = g[c] * act_slope<ACT>(fmaf(n, w[c], bias[c]));
        s1[c] += du;
        s2[c] = fmaf(du, n, s2[c]);
      }
    });
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    s_1[threadIdx.x][c] = s1[c];
    s_2[threadIdx.x][c] = s2[c];
  }
  for (int half = p.half; half >= 1; half /= 2) {
    __syncthreads();
    const int from = threadIdx.x + half * p.nb;
    if (q.ty < half && q.ty + half < q.step) {
#pragma unroll
      for (int c = 0; c < V; ++c) {
        s_1[threadIdx.x][c] += s_1[from][c];
        s_2[threadIdx.x][c] += s_2[from][c];
      }
    }
  }
  if (q.in && q.ty == 0) {
#pragma unroll
    for (int c = 0; c < V; ++c) s1[c] = s_1[threadIdx.x][c], s2[c] = s_2[threadIdx.x][c];
    float* to = p.part + (q.b * p.blocks + q.block) * 2 * a.C + q.c;
    store_n<float, V, false>(to, V, s1);
    store_n<float, V, false>(to + a.C, V, s2);
  }
}

// A clip's channels over its blocks, and the group's two means.  A channel has 256 / cg lanes, which take the blocks in
// turn; their sums are added in order.  JOINED: the channels' sums are there already.
template <bool JOINED>
__global__ void __launch_bounds__(256) norm_grad_join_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  __shared__ float s[4], s_1[256], s_2[256];
  const int g = blockIdx.x % (int)a.G, b = blockIdx.x / (int)a.G, cg = (int)(a.C / a.G);
  const int wide = std::min(cg, 256), lanes = 256 / wide, lane = threadIdx.x / wide, col = threadIdx.x % wide;
  const int64_t own = own_of(p, b);
  const float total = (float)own * (float)cg;
  float q1 = 0.0f, q2 = 0.0f;
  for (int i = col; i - col < cg; i += wide) {
    const int64_t c = (int64_t)g * cg + i;
    float s1 = 0.0f, s2 = 0.0f;
    if (!JOINED && i < cg && lane < lanes) {
      const float* part = p.part + (int64_t)b * p.blocks * 2 * a.C + c;
#pragma unroll 4
      for (int k = lane; k < p.blocks; k += lanes) {
        s1 += part[(int64_t)k * 2 * a.C];
        s2 += part[(int64_t)k * 2 * a.C + a.C];
      }
    }
    if (!JOINED) {
      __syncthreads();
      s_1[threadIdx.x] = s1;
      s_2[threadIdx.x] = s2;
      __syncthreads();
    }
    if (i < cg && lane == 0) {
      float* chan = p.chan + (int64_t)b * 2 * a.C + c;
      if (JOINED) {
        s1 = chan[0];
        s2 = chan[a.C];
      } else {
        for (int k = 1; k < lanes; ++k) {
          s1 += s_1[k * wide + col];
          s2 += s_2[k * wide + col];
        }
        chan[0] = s1;
        chan[a.C] = s2;
      }
      const float w = a.weight ? a.weight[c] : 1.0f;
      q1 = fmaf(w, s1, q1);
      q2 = fmaf(w, s2, q2);
    }
  }
  q1 = block_sum(q1, s);
  q2 = block_sum(q2, s);
  if (threadIdx.x == 0) {
    p.gsum[((int64_t)b * a.G + g) * 2] = own > 0 ? q1 / total : 0.0f;
    p.gsum[((int64_t)b * a.G + g) * 2 + 1] = own > 0 ? q2 / total : 0.0f;
  }
}

// dw and db: the clips' channels.
__global__ void __launch_bounds__(1024) norm_param_kernel(const NormParams p, int64_t rows, int64_t step) {
  const sed_norm_args& a = p.a;
  const int64_t c = (int64_t)blockIdx.x * kColumns + threadIdx.x % kColumns;
  const float v = column_sum(p.chan + c, rows, step, c < 2 * a.C);
  if (threadIdx.x >= kColumns || c >= 2 * a.C) return;
  if (c < a.C) {
    if (a.db) a.db[c] = v;
  } else if (a.dw) {
    a.dw[c - a.C] = v;
  }
}

template <class T, int V, bool VEC, int ACT>
__global__ void __launch_bounds__(256) norm_grad_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  const Cell q = cell<V, true>(p);
  if (!q.in) return;
  float mean[V], rstd[V], w[V], bias[V], m1[V], m2[V];
  channels<V>(p, q, mean, rstd, w, bias);
  each_group<V>(p, q, [&](int c, int64_t g) {
    m1[c] = p.gsum[g * 2];
    m2[c] = p.gsum[g * 2 + 1];
  });
  // dx = rstd (du w - m1 - n m2)
  float wr[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    wr[c] = w[c] * rstd[c];
    m1[c] *= rstd[c];
    m2[c] *= rstd[c];
  }
  const int64_t at = q.b * p.S * a.C + q.c;
  const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at;
  T* dx = static_cast<T*>(a.dx) + at;
  walk_two<T, V, grad_rows<ACT>(V)>(x, dy, q.r0 + q.ty, q.r1, q.step, a.C, [&](const float(&v)[V], const float(&g)[V], int64_t r) {
    float d[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float n = (v[c] - mean[c]) * rstd[c], du = g[c] * act_slope<ACT>(fmaf(n, w[c], bias[c]));
      d[c] = fmaf(-n, m2[c], fmaf(du, wr[c], -m1[c]));
    }
    store_n<T, V, VEC>(dx + r * a.C, V, d);
  });
  const float zero[V] = {};
  for (int64_t r = q.z0 + q.ty; r < q.z1; r += q.step) store_n<T, V, VEC>(dx + r * a.C, V, zero);
}

// The gradient of such a group in one launch: both maps' rows are read once; the channels' sums of du and du n go over the places in
// pairs through LDS, their weighted sums over the channels to all.  512 x 100 x 256 bf16 42 us (four launches of the walks 66), 2000 x 200 x 256 bf16 in 8 groups 178 us
// for 614 MB (232).
template <class T, int V, int HELD, int ACT>
__global__ void __launch_bounds__(1024) norm_whole_grad_kernel(const NormParams p) {
  const sed_norm_args& a = p.a;
  typedef T vt __attribute__((ext_vector_type(V)));
  extern __shared__ float sums[];  // [threads][V + 1]
  __shared__ float s[2][16];
  const unsigned item = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  if (item >= a.B * a.G) return;
  const int b = item / (unsigned)a.G, g = item % (unsigned)a.G, cg = (int)(a.C / a.G);
  const int nv = cg / V, tx = threadIdx.x % nv, ty = threadIdx.x / nv, step = blockDim.x / nv, waves = (blockDim.x + 63) / 64;
  const int own = (int)own_of(p, b), mine = ty < step ? own : 0;
  const int64_t c = g * cg + tx * V, at = b * p.S * a.C + c;
  const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at;
  T* dx = static_cast<T*>(a.dx) + at;
  vt v[HELD], e[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int r = ty + h * step;
    if (r < mine) {
      v[h] = *reinterpret_cast<const vt*>(x + r * a.C);
      e[h] = *reinterpret_cast<const vt*>(dy + r * a.C);
    }
  }
  const float mean = a.mean[item], rstd = a.rstd[item];
  float w[V], s1[V], s2[V], du[HELD][V];
  {
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[i] = a.weight ? a.weight[c + i] : 1.0f;
      bias[i] = a.bias ? a.bias[c + i] : 0.0f;
      s1[i] = s2[i] = 0.0f;
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (ty + h * step < mine)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = ((float)v[h][i] - mean) * rstd;
          du[h][i] = (float)e[h][i] * act_slope<ACT>(fmaf(n, w[i], bias[i]));
          s1[i] += du[h][i];
          s2[i] = fmaf(du[h][i], n, s2[i]);
        }
  }
  // over the places: lane (tx, 0) gets its channels' sums
  float(*const rows)[V + 1] = reinterpret_cast<float(*)[V + 1]>(sums);
  const auto over_places = [&](float (&t)[V]) {
    int half = 1;
    while (2 * half < step) half *= 2;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) rows[threadIdx.x][i] = t[i];
    for (; half >= 1; half /= 2) {
      __syncthreads();
      if (ty < half && ty + half < step)
#pragma unroll
        for (int i = 0; i < V; ++i) rows[threadIdx.x][i] += rows[threadIdx.x + half * nv][i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = rows[threadIdx.x][i];
  };
  over_places(s1);
  over_places(s2);
  float q1 = 0.0f, q2 = 0.0f;
  if (ty == 0) {
    float* chan = p.chan + (int64_t)b * 2 * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      chan[i] = s1[i];
      chan[a.C + i] = s2[i];
      q1 = fmaf(w[i], s1[i], q1);
      q2 = fmaf(w[i], s2[i], q2);
    }
  }
  q1 = wave_sum(q1);
  q2 = wave_sum(q2);
  if (threadIdx.x % 64 == 0) {
    s[0][threadIdx.x / 64] = q1;
    s[1][threadIdx.x / 64] = q2;
  }
  __syncthreads();
  q1 = q2 = 0.0f;
  for (int i = 0; i < waves; ++i) {
    q1 += s[0][i];
    q2 += s[1][i];
  }
  const float scale = own > 0 ? rstd / ((float)own * (float)cg) : 0.0f;
  q1 *= scale;
  q2 *= scale;
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] *= rstd;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int r = ty + h * step;
    if (r < mine) {
      float d[V];
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = fmaf(-((float)v[h][i] - mean) * rstd, q2, fmaf(du[h][i], w[i], -q1));
      store_n<T, V, true>(dx + r * a.C, V, d);
    }
  }
  const float zero[V] = {};
  if (ty < step)
    for (int64_t r = own + ty; r < p.S; r += step) store_n<T, V, true>(dx + r * a.C, V, zero);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_args(const sed_norm_args* a) {
  if (!a || a->B < 0 || a->T < 0 || a->F < 1 || a->C < 1 || a->G < 1 || a->C % a->G || !(a->eps >= 0.0f)) return SED_ERR_BAD_ARG;
  if (a->dtype != SED_F32 && a->dtype != SED_BF16 && a->dtype != SED_F16) return SED_ERR_BAD_ARG;
  if (a->act < SED_ACT_NONE || a->act > SED_ACT_GELU) return SED_ERR_BAD_ARG;
  if (a->B > 0 && a->T > 0 && (!a->x || !a->mean || !a->rstd)) return SED_ERR_BAD_ARG;
  if (a->B > 65535 || a->C > (1 << 19)) return SED_ERR_CAPACITY;
  return SED_OK;
}

struct Layout {
  int64_t part, chan, gsum, total;
  int32_t blocks, late;
};
// Blocks of a clip: 2048 over the batch, eight for each compute unit (4096 cost the joining kernels more than they gave the others);
// no more than one for every 32 places and 4096 values of the padded length (rounded up), so that its sums cost little beside its rows.  A
// clip's own places are divided evenly among them: a short clip's blocks may have one place or none.  The second walk leaves no sums:
// 8192 blocks, which end closer together (32 x 1001 x 64 x 64 forward and gradient: 435 us with 2048, 429 with 4096, 423 with 8192,
// 450 with 16384; fewer than 32 places each: 64 clips of up to 862 x 768 in 72 us, 57 with 32).
Layout layout_of(int64_t B, int64_t S, int64_t C, int64_t G) {
  Layout l{};
  const int64_t least = std::max<int64_t>(32, 4096 / C);
  const auto blocks = [&](int64_t most) { return (int32_t)std::max<int64_t>(1, std::min<int64_t>((S + least - 1) / least, most / std::max<int64_t>(1, B))); };
  l.blocks = blocks(kBlocks);
  l.late = blocks(8192);
  int64_t at = 0;
  const auto take = [&](int64_t k) { const int64_t o = at; at += (k + 63) / 64 * 64; return o; };
  l.part = take(B * l.blocks * 2 * C);
  l.chan = take(B * 2 * C);
  l.gsum = take(B * G * 2);
  l.total = at;
  return l;
}

// Threads of norm_whole_kernel (BACK: of norm_whole_grad_kernel) for lanes of V channels and `held` rows, or 0 where it does not fit
// or is slower: 8 rows a lane (more registers, more code) beyond a workgroup a compute unit (64 x 862 x 768 bf16: 71 us, the walks 68;
// 16 x 101 x 64 x 32 fp32 15 us, 17); pieces of lines under 32 bytes where more than 96 MiB are read (4 channels a group of 256 x 101 x
// 32 x 32: fp32 62 us, the walks 57, bf16 gradient 106, 73; but 64 x 125 x 16 x 64 fp32 23, 28 and gradient 37, 44).  The border lies
// right under what was measured slower (98 MiB and more; up to 73 MiB was faster), too high for bf16 gradients: 1960 x 200 x 64 in 8
// groups takes 183 us forward and gradient, 2000 clips of it by the walks 144.  Many groups: as few threads as hold one, so that a
// compute unit has several; else all, for the shortest way through.
int whole_threads(const NormParams& p, int V, int held, bool back) {
  const sed_norm_args& a = p.a;
  const int64_t cg = a.C / a.G, nv = cg / V, items = a.B * a.G;
  if (cg % V || nv > 1024 || p.S > held * (1024 / nv)) return 0;
  if (held > 4 && items > 256) return 0;
  const int64_t size = a.dtype == SED_F32 ? 4 : 2;
  if (cg * size < 32 && a.B * p.S * a.C * size * (back ? 2 : 1) > (96 << 20)) return 0;
  int threads = 1024;
  if (items >= 512)
    while (threads > 256 && nv <= threads / 2 && p.S <= held * (threads / 2 / nv)) threads /= 2;
  threads = (int)std::min<int64_t>(threads, (p.S * nv + 63) / 64 * 64);
  return grid_fits(items + 7, threads) ? threads : 0;
}

template <class T, int V, int HELD, int ACT>
int launch_whole(const NormParams& p, int threads, hipStream_t s) {
  const int64_t grid = (p.a.B * p.a.G + 7) / 8 * 8;
  norm_whole_kernel<T, V, HELD, ACT><<<(unsigned)grid, threads, 0, s>>>(p);
  return seq_status(hipGetLastError());
}

int launch_param(const NormParams& p, hipStream_t s) {
  const sed_norm_args& a = p.a;
  if (a.dw || a.db) {
    int64_t rows = a.B, step = 2 * a.C;
    fold_rows(p.chan, rows, step, 2 * a.C, s);
    norm_param_kernel<<<(unsigned)((2 * a.C + kColumns - 1) / kColumns), 1024, 0, s>>>(p, rows, step);
  }
  return seq_status(hipGetLastError());
}

template <class T, int V, int ACT>
int launch_whole_grad(const NormParams& p, int threads, hipStream_t s) {
  const int64_t grid = (p.a.B * p.a.G + 7) / 8 * 8;
  norm_whole_grad_kernel<T, V, 4, ACT><<<(unsigned)grid, threads, threads * (V + 1) * 4, s>>>(p);
  return launch_param(p, s);
}

template <class T, int V, bool VEC, int ACT>
int launch(const NormParams& p, bool back, hipStream_t s) {
  const sed_norm_args& a = p.a;
  if constexpr (VEC) {
    if (!back) {
      if (const int n = whole_threads(p, V, 4, false)) return launch_whole<T, V, 4, ACT>(p, n, s);
      if (const int n = whole_threads(p, V, 8, false)) return launch_whole<T, V, 8, ACT>(p, n, s);
      if constexpr (V == 8) {
        if (const int n = whole_threads(p, 4, 4, false)) return launch_whole<T, 4, 4, ACT>(p, n, s);
        if (const int n = whole_threads(p, 4, 8, false)) return launch_whole<T, 4, 8, ACT>(p, n, s);
      }
    } else {
      if (const int n = whole_threads(p, V, 4, true)) return launch_whole_grad<T, V, ACT>(p, n, s);
      if constexpr (V == 8)
        if (const int n = whole_threads(p, 4, 4, true)) return launch_whole_grad<T, 4, ACT>(p, n, s);
    }
  }
  if (!grid_fits(a.B * a.G, 256)) return SED_ERR_CAPACITY;  // of the joins
  const dim3 grid((unsigned)p.blocks, (unsigned)a.B, (unsigned)((p.nv + p.nb - 1) / p.nb)), late((unsigned)p.late, grid.y, grid.z);
  // more blocks and channels a group than a workgroup joins in 8 steps: a launch of its own for the blocks
  const int64_t cg = a.C / a.G;
  const bool far = p.blocks * cg > 8 * 256, many = far && p.blocks > 1;
  const dim3 channels((unsigned)((a.C + 15) / 16), grid.y);
  const unsigned groups = (unsigned)(a.B * a.G), threads = (unsigned)((256 / p.nb * p.nb + 63) / 64 * 64);
  if (!back) {
    norm_stats_kernel<T, V, VEC><<<grid, threads, 0, s>>>(p);
    if (!far) {
      norm_join_kernel<8, false><<<groups, 256, 0, s>>>(p);
    } else {
      if (many) norm_channel_kernel<false><<<channels, 1024, 0, s>>>(p);
      if (cg <= 8 * 256)
        norm_join_kernel<8, true><<<groups, 256, 0, s>>>(p);
      else
        norm_join_kernel<0, true><<<groups, 256, 0, s>>>(p);
    }
    norm_apply_kernel<T, V, VEC, ACT><<<late, threads, 0, s>>>(p);
  } else {
    norm_grad_sums_kernel<T, V, VEC, ACT><<<grid, threads, 0, s>>>(p);
    if (!many) {
      norm_grad_join_kernel<false><<<groups, 256, 0, s>>>(p);
    } else {
      norm_channel_kernel<true><<<channels, 1024, 0, s>>>(p);
      norm_grad_join_kernel<true><<<groups, 256, 0, s>>>(p);
    }
    norm_grad_kernel<T, V, VEC, ACT><<<late, threads, 0, s>>>(p);
    return launch_param(p, s);
  }
  return seq_status(hipGetLastError());
}

template <class T, int V, bool VEC>
int go_act(const NormParams& p, bool back, hipStream_t s) {
  switch (p.a.act) {
    case SED_ACT_SILU: return launch<T, V, VEC, SED_ACT_SILU>(p, back, s);
    case SED_ACT_RELU: return launch<T, V, VEC, SED_ACT_RELU>(p, back, s);
    case SED_ACT_GELU: return launch<T, V, VEC, SED_ACT_GELU>(p, back, s);
    default: return launch<T, V, VEC, SED_ACT_NONE>(p, back, s);
  }
}

int run(const sed_norm_args* args, bool back, void* stream) {
  NormParams p{};
  p.a = *args;
  sed_norm_args& a = p.a;
  p.S = a.T * a.F;
  const Layout l = layout_of(a.B, p.S, a.C, a.G);
  if (!a.ws || a.ws_bytes < l.total * 4 || !aligned(a.ws, 16)) return SED_ERR_CAPACITY;
  const int V = a.dtype == SED_F32 ? 4 : 8;
  const bool vec = a.C % V == 0 && aligned(a.x, 16) && aligned(a.y, 16) && aligned(a.dy, 16) && aligned(a.dx, 16);
  p.nv = (int32_t)(vec ? a.C / V : a.C);
  p.nb = std::min(p.nv, 256);
  if ((p.nv + p.nb - 1) / p.nb > 65535) return SED_ERR_CAPACITY;
  p.half = 0;
  for (int lanes = 256 / p.nb, h = 1; h < lanes; h *= 2) p.half = h;
  p.blocks = l.blocks;
  p.late = l.late;
  float* ws = static_cast<float*>(a.ws);
  p.part = ws + l.part;
  p.chan = ws + l.chan;
  p.gsum = ws + l.gsum;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == SED_F32) return vec ? go_act<float, 4, true>(p, back, s) : go_act<float, 1, false>(p, back, s);
  if (a.dtype == SED_BF16) return vec ? go_act<bf16, 8, true>(p, back, s) : go_act<bf16, 1, false>(p, back, s);
  return vec ? go_act<f16, 8, true>(p, back, s) : go_act<f16, 1, false>(p, back, s);
}

}  // namespace
}  // namespace sed

extern "C" int64_t sed_group_norm_workspace(int64_t B, int64_t T, int64_t F, int64_t C, int64_t G) {
  if (B < 0 || T < 0 || F < 1 || C < 1 || G < 1 || C % G) return SED_ERR_BAD_ARG;
  return sed::layout_of(B, T * F, C, G).total * 4;
}

extern "C" int sed_group_norm_forward(const sed_norm_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->T == 0) return SED_OK;
  if (!args->y) return SED_ERR_BAD_ARG;
  return sed::run(args, false, stream);
}

extern "C" int sed_group_norm_backward(const sed_norm_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->T == 0) return SED_OK;
  if (!args->dy || !args->dx) return SED_ERR_BAD_ARG;
  return sed::run(args, true, stream);
}
