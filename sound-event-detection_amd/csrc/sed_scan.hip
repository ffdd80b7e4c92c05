// Gated linear recurrence along the frames of a clip, its gradient and its one-frame form, for gfx950.
//
//   delta_t[d] = softplus(dt_t[d] + dt_bias[d])   (or dt + dt_bias)
//   h_t[d,n]   = exp(delta_t[d] A[d,n]) h_{t-1}[d,n] + delta_t[d] x_t[d] B_t[g,n]
//   y_t[d]     = (sum_n C_t[g,n] h_t[d,n] + skip[d] x_t[d]) * silu(z_t[d])
//
// Bound: the vector unit.  A state takes one exp2 and four multiply-adds per frame and no matrix instruction helps, since the
// decay differs per channel, state and frame.  So the layout serves the vector unit: one wave per workgroup, every lane holds
// 4 channels x NS states in registers and walks along the frames, SPLIT lanes share a channel's NP = NS * SPLIT states.
// B and C are then read from LDS once for 4 channels, the sum over states is NS multiply-adds and a few lane exchanges for 4
// channels at once, and in the gradient the sum over channels is 4 multiply-adds in the lane before any exchange.
// Frames come in tiles of TT rows: the lanes load a tile's rows (each row once), form delta and delta * x in LDS, scan, and
// write the finished rows, while the next tile's rows are on their way.
//
// A clip is cut into chunks where there are too few waves to fill the card: a first pass gives every chunk's own end state
// from zero and the sum of its delta (the decay over a chunk is exp(A * sum), no product of decays is kept), chunk_join_kernel
// runs over the chunks, and the main pass starts each chunk from its state.  The gradient is the same recurrence from the
// other end: g_t = C_t gy_t + exp(delta_{t+1} A) g_{t+1}.  It recomputes a tile's states from the state in front of the
// tile, which the forward pass keeps (`saved`), and keeps exp(delta A) h_{t-1} of the tile's TT frames in registers.
// States, decays and sums are fp32; x, dt, z, B, C, y and their gradients are fp32, bf16 or fp16, rounded once at the store.
#include "seq_core.h"

#include <algorithm>

namespace sed {
namespace {

struct ScanParams {
  sed_scan_args a;
  int64_t L_chunk;  // frames of a chunk, a multiple of TT
  int32_t K;        // chunks
  int32_t tiles;    // channel tiles of a group
  int32_t saved_n;  // ceil(L / TT)
  float* chunk_h;   // [B][K][NP][D]  end states from zero, then the states in front of the chunks
  float* chunk_s;   // [B][K][D]      sums of delta
  float* part_bc;   // [B][G * tiles][L][2 * NP]  dB, dC of one wave's channels
  float* part_a;    // [B * K][D * NP] dA  [NP][D] per row
  float* part_d;    // [B * K][2][D]  d skip, d dt_bias
};

// Tile geometry of one instance.
template <int NS, int SPLIT>
struct Geo {
  static constexpr int NP = NS * SPLIT;       // states, padded
  static constexpr int J = 64 / SPLIT;        // lanes along channels
  static constexpr int CW = 4 * J;            // channels of a wave
  static constexpr int TT = NS == 8 ? 4 : 8;  // frames of a tile: TT * 4 * NS = 128 registers hold a tile's states (fewer with NS < 4)
  static constexpr int R = TT / SPLIT;        // rows a lane loads
  static constexpr int PB = (TT * NP + 63) / 64;
  static_assert(R * SPLIT == TT, "");
};

// Where a wave works.
struct Where {
  int b, chunk, g, s, j;
  int64_t own;       // frames of the clip's own
  int64_t c0;        // first channel of the lane
  int nc;            // channels of the lane (0..4)
  int tile;          // over all groups
};

template <class G>
__device__ __forceinline__ Where where(const ScanParams& p) {
  Where w;
  const sed_scan_args& a = p.a;
  const int all = p.tiles * a.G;
  unsigned i = blockIdx.x;
  w.tile = i % all;
  i /= all;
  w.chunk = i % p.K;
  w.b = i / p.K;
  w.g = w.tile / p.tiles;
  w.s = threadIdx.x / G::J;
  w.j = threadIdx.x % G::J;
  const int64_t cg = a.D / a.G, in = (int64_t)(w.tile % p.tiles) * G::CW + 4 * w.j;
  w.c0 = w.g * cg + in;
  w.nc = (int)std::max<int64_t>(0, std::min<int64_t>(4, cg - in));
  w.own = a.L;
  if (a.frames) w.own = std::max<int64_t>(0, std::min<int64_t>(a.L, a.frames[w.b]));
  return w;
}

// Row of the clip that comes i-th: behind the clip's own rows every row is itself.
__device__ __forceinline__ int64_t row_of(const ScanParams& p, int64_t own, int64_t i) {
  return p.a.reverse && i < own ? own - 1 - i : i;
}

// Rows of a tile as a lane loads them: 4 channels of rows i0 + r * SPLIT + s.
template <class G, class T, bool VEC>
__device__ __forceinline__ void load_rows(const ScanParams& p, const Where& w, const void* base, int64_t sb, int64_t st, int64_t i0,
                                          float (&out)[G::R][4]) {
#pragma unroll
  for (int r = 0; r < G::R; ++r) {
    const int64_t i = i0 + r * (64 / G::J) + w.s;
    const bool in = i < w.own;
    const T* q = static_cast<const T*>(base) + w.b * sb + (in ? row_of(p, w.own, i) : 0) * st + w.c0;
    load_n<T, 4, VEC>(q, in ? w.nc : 0, out[r]);
  }
}

// B or C of a tile: element e = lane + 64 i is state e % NP of row e / NP.
template <class G, class T>
__device__ __forceinline__ void load_bc(const ScanParams& p, const Where& w, const void* base, int64_t sb, int64_t st, int64_t sg, int64_t i0,
                                        float (&out)[G::PB]) {
#pragma unroll
  for (int q = 0; q < G::PB; ++q) {
    const int e = threadIdx.x + 64 * q, n = e % G::NP;
    const int64_t i = i0 + e / G::NP;
    const bool in = e < G::TT * G::NP && n < p.a.N && i < w.own;
    const T* at = static_cast<const T*>(base) + w.b * sb + (in ? row_of(p, w.own, i) : 0) * st + w.g * sg + (in ? n : 0);
    out[q] = in ? (float)*at : 0.0f;
  }
}
template <class G>
__device__ __forceinline__ void put_bc(const float (&v)[G::PB], float* to) {
#pragma unroll
  for (int q = 0; q < G::PB; ++q) {
    const int e = threadIdx.x + 64 * q;
    if (e < G::TT * G::NP) to[e] = v[q];
  }
}

template <int NS>
__device__ __forceinline__ void get_states(const float* from, float (&v)[NS]) {
  if constexpr (NS % 4 == 0) {
#pragma unroll
    for (int q = 0; q < NS / 4; ++q) {
      const f32x4 t = reinterpret_cast<const f32x4*>(from)[q];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = from[i];
  }
}

__device__ __forceinline__ void get4(const float* from, float (&v)[4]) {
  const f32x4 t = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = t[i];
}
__device__ __forceinline__ void put4(const float (&v)[4], float* to) {
  *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
}

// Sums of v[4] over the SPLIT lanes that share a channel; afterwards lane s of a channel group holds, for SPLIT = 4, channel s
// (out[0]); for SPLIT = 2, channels s and 2 + s... as `put_sums` writes them.
template <int SPLIT, int CW>
__device__ __forceinline__ void put_sums(const float (&v)[4], int s, int j, float* row) {
  if constexpr (SPLIT == 4) {
    // rows of 16 lanes s = 0..3: halves first (channels 0 | 2 and 1 | 3), then neighbouring rows
    const float lo = fold32(v[0], v[2]), hi = fold32(v[1], v[3]);
    row[4 * j + s] = fold16(lo, hi);
  } else if constexpr (SPLIT == 2) {
    const float a = fold32(v[0], v[2]), b = fold32(v[1], v[3]);
    *reinterpret_cast<f32x2*>(row + 4 * j + 2 * s) = f32x2{a, b};
  } else {
    put4(v, row + 4 * j);
  }
}

// states of a lane from / to a [NP][D] plane
template <class G, int NS, bool VEC>
__device__ __forceinline__ void load_plane(const float* plane, int64_t D, const Where& w, float (&h)[4][NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    float v[4];
    load_n<float, 4, VEC>(plane + (int64_t)(w.s * NS + n) * D + w.c0, w.nc, v);
#pragma unroll
    for (int c = 0; c < 4; ++c) h[c][n] = v[c];
  }
}
template <class G, int NS, bool VEC>
__device__ __forceinline__ void store_plane(float* plane, int64_t D, const Where& w, const float (&h)[4][NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = h[c][n];
    store_n<float, 4, VEC>(plane + (int64_t)(w.s * NS + n) * D + w.c0, w.nc, v);
  }
}
// states of a lane from / to the caller's [D][N]
template <class G, int NS>
__device__ __forceinline__ void load_dn(const float* base, int N, const Where& w, float (&h)[4][NS]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int k = w.s * NS + n;
      h[c][n] = c < w.nc && k < N ? base[(w.c0 + c) * N + k] : 0.0f;
    }
}
template <class G, int NS>
__device__ __forceinline__ void store_dn(float* base, int N, const Where& w, const float (&h)[4][NS]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int k = w.s * NS + n;
      if (c < w.nc && k < N) base[(w.c0 + c) * N + k] = h[c][n];
    }
}

__device__ __forceinline__ float delta_of(const ScanParams& p, float v) { return p.a.softplus ? softplus(v) : v; }

__device__ __forceinline__ void per_channel(const float* from, const Where& w, float (&v)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = from && c < w.nc ? from[w.c0 + c] : 0.0f;
}

// ---- forward ------------------------------------------------------------------------------------------------------------

// ENDS: only the chunk's end state from zero and its sum of delta.  Otherwise the chunk's outputs.
template <int NS, int SPLIT, class T, bool VEC, bool ENDS>
__global__ void __launch_bounds__(64) scan_forward_kernel(const ScanParams p) {
  using G = Geo<NS, SPLIT>;
  const sed_scan_args& a = p.a;
  const Where w = where<G>(p);
  __shared__ __attribute__((aligned(16))) float s_dl[G::TT][G::CW], s_dx[G::TT][G::CW], s_y[ENDS ? 1 : G::TT][G::CW];
  __shared__ __attribute__((aligned(16))) float s_B[G::TT][G::NP], s_C[G::TT][G::NP];
  const int64_t begin = w.chunk * p.L_chunk, end = std::min<int64_t>(begin + p.L_chunk, a.L);
  if (ENDS && (w.chunk == p.K - 1 || begin >= w.own)) return;  // chunk_join_kernel reads no such chunk

  float A2[4][NS], h[4][NS], bias[4], skip[4], sum[4] = {0, 0, 0, 0};
  load_dn<G, NS>(a.A, a.N, w, A2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) A2[c][n] *= kLog2e;
  per_channel(a.dt_bias, w, bias);
  per_channel(a.skip, w, skip);
  if (!ENDS && p.K > 1 && begin < w.own) {
    load_plane<G, NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, h);
  } else if (!ENDS && a.h0) {
    load_dn<G, NS>(a.h0 + (int64_t)w.b * a.D * a.N, a.N, w, h);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < NS; ++n) h[c][n] = 0.0f;
  }

  float x[G::R][4], dt[G::R][4], z[G::R][4], bv[G::PB], cv[G::PB];
  const auto fetch = [&](int64_t i0) {
    load_rows<G, T, VEC>(p, w, a.x, a.x_b, a.x_t, i0, x);
    load_rows<G, T, VEC>(p, w, a.dt, a.dt_b, a.dt_t, i0, dt);
    load_bc<G, T>(p, w, a.Bm, a.Bm_b, a.Bm_t, a.Bm_g, i0, bv);
    if (!ENDS) {
      if (a.z) load_rows<G, T, VEC>(p, w, a.z, a.z_b, a.z_t, i0, z);
      load_bc<G, T>(p, w, a.Cm, a.Cm_b, a.Cm_t, a.Cm_g, i0, cv);
    }
  };
  fetch(begin);
  for (int64_t i0 = begin; i0 < end; i0 += G::TT) {
    const bool live = i0 < w.own;
    float xs[G::R][4], zs[G::R][4];
    if (live) {
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        const bool in = i0 + r * SPLIT + w.s < w.own;
        float dl[4], dx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          dl[c] = in ? delta_of(p, dt[r][c] + bias[c]) : 0.0f;
          dx[c] = in ? dl[c] * x[r][c] : 0.0f;
          if (ENDS) sum[c] += dl[c];
          xs[r][c] = x[r][c];
          zs[r][c] = z[r][c];
        }
        put4(dl, &s_dl[r * SPLIT + w.s][4 * w.j]);
        put4(dx, &s_dx[r * SPLIT + w.s][4 * w.j]);
      }
      put_bc<G>(bv, &s_B[0][0]);
      if (!ENDS) put_bc<G>(cv, &s_C[0][0]);
      if (!ENDS && a.saved) store_plane<G, NS, VEC>(a.saved + ((int64_t)w.b * p.saved_n + i0 / G::TT) * G::NP * a.D, a.D, w, h);
      if (i0 + G::TT < end) fetch(i0 + G::TT);
      __syncthreads();
#pragma unroll
      for (int t = 0; t < G::TT; ++t) {
        float dl[4], dx[4], B[NS], C[NS], y[4];
        get4(&s_dl[t][4 * w.j], dl);
        get4(&s_dx[t][4 * w.j], dx);
        get_states<NS>(&s_B[t][w.s * NS], B);
        if (!ENDS) get_states<NS>(&s_C[t][w.s * NS], C);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          y[c] = 0.0f;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            h[c][n] = fmaf(exp2_hw(dl[c] * A2[c][n]), h[c][n], dx[c] * B[n]);
            if (!ENDS) y[c] = fmaf(C[n], h[c][n], y[c]);
          }
        }
        if (!ENDS) put_sums<SPLIT, G::CW>(y, w.s, w.j, &s_y[t][0]);
      }
      __syncthreads();
    }
    if (!ENDS) {
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        const int64_t i = i0 + r * SPLIT + w.s;
        float y[4] = {0, 0, 0, 0};
        if (i < w.own) {
          get4(&s_y[r * SPLIT + w.s][4 * w.j], y);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            y[c] = fmaf(skip[c], xs[r][c], y[c]);
            if (a.z) y[c] *= zs[r][c] * sigmoid(zs[r][c]);
          }
        }
        if (i < end)
          store_n<T, 4, VEC>(static_cast<T*>(a.y) + ((int64_t)w.b * a.L + row_of(p, w.own, i)) * a.D + w.c0, w.nc, y);
      }
      __syncthreads();
    }
  }
  if (ENDS) {
    store_plane<G, NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, h);
    // every lane of a channel summed its own rows
    __syncthreads();
    put_sums<SPLIT, G::CW>(sum, w.s, w.j, &s_dl[0][0]);
    __syncthreads();
    if (w.s == 0) {
      float v[4];
      get4(&s_dl[0][4 * w.j], v);
      store_n<float, 4, VEC>(p.chunk_s + ((int64_t)w.b * p.K + w.chunk) * a.D + w.c0, w.nc, v);
    }
  } else if (a.h_last && (w.own > 0 ? begin < w.own && w.own <= begin + p.L_chunk : w.chunk == 0)) {
    store_dn<G, NS>(a.h_last + (int64_t)w.b * a.D * a.N, a.N, w, h);
  }
}

// The states in front of the chunks, over the chunks in order (BACK: the gradients behind them, from the last).  One thread
// per channel and state.  In: every chunk's end state from zero; out, in its place: the state it starts from.
template <bool BACK>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ScanParams p, int NP) {
  const sed_scan_args& a = p.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * NP * a.D) return;
  const int64_t d = i % a.D, n = i / a.D % NP, b = i / a.D / NP;
  int64_t own = a.L;
  if (a.frames) own = std::max<int64_t>(0, std::min<int64_t>(a.L, a.frames[b]));
  const int k_own = (int)((own + p.L_chunk - 1) / p.L_chunk);
  const bool real = n < a.N;
  const float A2 = real ? a.A[d * a.N + n] * kLog2e : 0.0f;
  const float* first = BACK ? a.dh_last : a.h0;
  float h = first && real ? first[(b * a.D + d) * a.N + n] : 0.0f;
  float* hp = p.chunk_h + ((int64_t)b * p.K * NP + n) * a.D + d;
  const float* sp = p.chunk_s + (int64_t)b * p.K * a.D + d;
#pragma unroll 4
  for (int q = 0; q < k_own; ++q) {
    const int k = BACK ? k_own - 1 - q : q;
    const float end = q < k_own - 1 ? hp[(int64_t)k * NP * a.D] : 0.0f, s = q < k_own - 1 ? sp[(int64_t)k * a.D] : 0.0f;
    hp[(int64_t)k * NP * a.D] = h;
    h = fmaf(exp2_hw(A2 * s), h, end);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------

// 2 NS values v over the J lanes of a channel row; afterwards `value` is the sum of v[index] in the lanes where `write` holds.
template <int NV, int J>
__device__ __forceinline__ void sum_lanes(float (&v)[NV], int j, float& value, int& index, bool& write) {
  int n = NV;
  index = 0;
  write = true;
#pragma unroll
  for (int bit = J / 2; bit >= 1; bit /= 2) {
    const bool up = j & bit;
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i)
        if (i < n) {
          if (bit == 32) v[i] = fold32(v[i], v[i + n]);
          if (bit == 16) v[i] = fold16(v[i], v[i + n]);
          if (bit < 16) {
            const float lo = bit == 8 ? v[i] + dpp<kRor8>(v[i]) : bit == 4 ? v[i] + dpp<kHalfMirror>(v[i]) : bit == 2 ? v[i] + dpp<kXor2>(v[i]) : v[i] + dpp<kXor1>(v[i]);
            const float hi = bit == 8 ? v[i + n] + dpp<kRor8>(v[i + n]) : bit == 4 ? v[i + n] + dpp<kHalfMirror>(v[i + n])
                             : bit == 2 ? v[i + n] + dpp<kXor2>(v[i + n]) : v[i + n] + dpp<kXor1>(v[i + n]);
            v[i] = up ? hi : lo;
          }
        }
      if (up) index += n;
    } else {
      if (bit == 32) v[0] = fold32(v[0], v[0]);
      if (bit == 16) v[0] = fold16(v[0], v[0]);
      if (bit == 8) v[0] += dpp<kRor8>(v[0]);
      if (bit == 4) v[0] += dpp<kHalfMirror>(v[0]);
      if (bit == 2) v[0] += dpp<kXor2>(v[0]);
      if (bit == 1) v[0] += dpp<kXor1>(v[0]);
      write = write && !up;
    }
  }
  value = v[0];
}

// ENDS: only the gradient that reaches the frame in front of the chunk from the chunk's own outputs, and the sum of delta.
template <int NS, int SPLIT, class T, bool VEC, bool ENDS>
__global__ void __launch_bounds__(64) scan_backward_kernel(const ScanParams p) {
  using G = Geo<NS, SPLIT>;
  const sed_scan_args& a = p.a;
  const Where w = where<G>(p);
  constexpr int TX = ENDS ? 1 : G::TT;
  __shared__ __attribute__((aligned(16))) float s_dl[G::TT][G::CW], s_gy[G::TT][G::CW], s_dx[TX][G::CW];
  __shared__ __attribute__((aligned(16))) float s_y[TX][G::CW], s_1[TX][G::CW], s_2[TX][G::CW];
  __shared__ __attribute__((aligned(16))) float s_B[G::TT][G::NP], s_C[G::TT][G::NP];
  const int64_t begin = w.chunk * p.L_chunk, stop = std::min<int64_t>(begin + p.L_chunk, a.L), end = std::min<int64_t>(stop, w.own);
  if (ENDS && (w.chunk == 0 || begin >= w.own)) return;

  float A2[4][NS], g[4][NS], dA[4][NS], bias[4], skip[4], sum[4] = {0, 0, 0, 0}, dskip[4] = {0, 0, 0, 0}, dbias[4] = {0, 0, 0, 0};
  load_dn<G, NS>(a.A, a.N, w, A2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      A2[c][n] *= kLog2e;
      dA[c][n] = g[c][n] = 0.0f;
    }
  per_channel(a.dt_bias, w, bias);
  per_channel(a.skip, w, skip);
  // g: exp(delta_{t+1} A) g_{t+1}, what reaches frame t from behind
  if (!ENDS && begin < w.own) {
    if (p.K > 1)
      load_plane<G, NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, g);
    else if (a.dh_last)
      load_dn<G, NS>(a.dh_last + (int64_t)w.b * a.D * a.N, a.N, w, g);
  }
  if (!ENDS && w.own == 0 && a.dh_last) load_dn<G, NS>(a.dh_last + (int64_t)w.b * a.D * a.N, a.N, w, g);

  // rows behind the clip's own have no gradient
  if (!ENDS) {
    const float zero[4] = {0, 0, 0, 0};
    for (int64_t i = std::max<int64_t>(begin, w.own) + w.s; i < stop; i += SPLIT) {
      const int64_t at = ((int64_t)w.b * a.L + i) * a.D + w.c0;
      store_n<T, 4, VEC>(static_cast<T*>(a.dx) + at, w.nc, zero);
      store_n<T, 4, VEC>(static_cast<T*>(a.ddt) + at, w.nc, zero);
      if (a.dz) store_n<T, 4, VEC>(static_cast<T*>(a.dz) + at, w.nc, zero);
    }
  }

  float x[G::R][4], dt[G::R][4], z[G::R][4], dy[G::R][4], bv[G::PB], cv[G::PB];
  const auto fetch = [&](int64_t i0) {
    load_rows<G, T, VEC>(p, w, a.dt, a.dt_b, a.dt_t, i0, dt);
    load_rows<G, T, VEC>(p, w, a.dy, a.dy_b, a.dy_t, i0, dy);
    if (a.z) load_rows<G, T, VEC>(p, w, a.z, a.z_b, a.z_t, i0, z);
    load_bc<G, T>(p, w, a.Cm, a.Cm_b, a.Cm_t, a.Cm_g, i0, cv);
    if (!ENDS) {
      load_rows<G, T, VEC>(p, w, a.x, a.x_b, a.x_t, i0, x);
      load_bc<G, T>(p, w, a.Bm, a.Bm_b, a.Bm_t, a.Bm_g, i0, bv);
    }
  };
  const int64_t tiles = begin < end ? (end - begin + G::TT - 1) / G::TT : 0;
  if (tiles) fetch(begin + (tiles - 1) * G::TT);
  for (int64_t k = tiles - 1; k >= 0; --k) {
    const int64_t i0 = begin + k * G::TT;
    float h[4][NS];
    if (!ENDS) load_plane<G, NS, VEC>(a.saved + ((int64_t)w.b * p.saved_n + i0 / G::TT) * G::NP * a.D, a.D, w, h);
    float xs[G::R][4], dls[G::R][4], vs[G::R][4], zs[G::R][4], dys[G::R][4], gys[G::R][4];
#pragma unroll
    for (int r = 0; r < G::R; ++r) {
      const bool in = i0 + r * SPLIT + w.s < w.own;
      float dx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        vs[r][c] = dt[r][c] + bias[c];
        dls[r][c] = in ? delta_of(p, vs[r][c]) : 0.0f;
        dys[r][c] = dy[r][c];
        zs[r][c] = z[r][c];
        gys[r][c] = a.z ? dy[r][c] * z[r][c] * sigmoid(z[r][c]) : dy[r][c];
        if (!in) gys[r][c] = 0.0f;
        if (ENDS) sum[c] += dls[r][c];
        xs[r][c] = x[r][c];
        dx[c] = ENDS ? 0.0f : dls[r][c] * x[r][c];
        if (!in) dx[c] = 0.0f;
      }
      put4(dls[r], &s_dl[r * SPLIT + w.s][4 * w.j]);
      put4(gys[r], &s_gy[r * SPLIT + w.s][4 * w.j]);
      if (!ENDS) put4(dx, &s_dx[r * SPLIT + w.s][4 * w.j]);
    }
    put_bc<G>(cv, &s_C[0][0]);
    if (!ENDS) put_bc<G>(bv, &s_B[0][0]);
    if (k) fetch(i0 - G::TT);
    __syncthreads();
    float P[ENDS ? 1 : G::TT][4][NS];  // exp(delta_t A) h_{t-1}
    if (!ENDS) {
#pragma unroll
      for (int t = 0; t < G::TT; ++t) {
        float dl[4], dx[4], B[NS], C[NS], y[4];
        get4(&s_dl[t][4 * w.j], dl);
        get4(&s_dx[t][4 * w.j], dx);
        get_states<NS>(&s_B[t][w.s * NS], B);
        get_states<NS>(&s_C[t][w.s * NS], C);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          y[c] = 0.0f;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            P[t][c][n] = exp2_hw(dl[c] * A2[c][n]) * h[c][n];
            h[c][n] = fmaf(dx[c], B[n], P[t][c][n]);
            y[c] = fmaf(C[n], h[c][n], y[c]);
          }
        }
        put_sums<SPLIT, G::CW>(y, w.s, w.j, &s_y[t][0]);
      }
    }
#pragma unroll
    for (int t = G::TT - 1; t >= 0; --t) {
      float dl[4], gy[4], dx[4], B[NS], C[NS], S1[4], S2[4], v[2 * NS];
      get4(&s_dl[t][4 * w.j], dl);
      get4(&s_gy[t][4 * w.j], gy);
      get_states<NS>(&s_C[t][w.s * NS], C);
      if (!ENDS) {
        get4(&s_dx[t][4 * w.j], dx);
        get_states<NS>(&s_B[t][w.s * NS], B);
      }
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n) v[n] = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        S1[c] = S2[c] = 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const float gt = fmaf(C[n], gy[c], g[c][n]);
          if (!ENDS) {
            const float gp = gt * P[t][c][n];
            v[n] = fmaf(gt, dx[c], v[n]);
            v[NS + n] = fmaf(gy[c], fmaf(dx[c], B[n], P[t][c][n]), v[NS + n]);
            S1[c] = fmaf(gt, B[n], S1[c]);
            S2[c] = fmaf(gp, A2[c][n], S2[c]);
            dA[c][n] = fmaf(gp, dl[c], dA[c][n]);
          }
          g[c][n] = exp2_hw(dl[c] * A2[c][n]) * gt;
        }
      }
      if (!ENDS) {
        put_sums<SPLIT, G::CW>(S1, w.s, w.j, &s_1[t][0]);
        put_sums<SPLIT, G::CW>(S2, w.s, w.j, &s_2[t][0]);
        float value;
        int index;
        bool write;
        sum_lanes<2 * NS, G::J>(v, w.j, value, index, write);
        const int64_t i = i0 + t;
        if (write && i < w.own) {
          const int at = index < NS ? w.s * NS + index : G::NP + w.s * NS + index - NS;
          p.part_bc[(((int64_t)w.b * p.tiles * a.G + w.tile) * a.L + row_of(p, w.own, i)) * (2 * G::NP) + at] = value;
        }
      }
    }
    __syncthreads();
    if (!ENDS) {
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        const int64_t i = i0 + r * SPLIT + w.s;
        if (i < w.own) {
          float y[4], s1[4], s2[4], dx[4], ddt[4], dz[4];
          get4(&s_y[r * SPLIT + w.s][4 * w.j], y);
          get4(&s_1[r * SPLIT + w.s][4 * w.j], s1);
          get4(&s_2[r * SPLIT + w.s][4 * w.j], s2);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            dx[c] = fmaf(dls[r][c], s1[c], skip[c] * gys[r][c]);
            ddt[c] = fmaf(xs[r][c], s1[c], kLn2 * s2[c]);
            if (a.softplus) ddt[c] *= sigmoid(vs[r][c]);
            dskip[c] = fmaf(gys[r][c], xs[r][c], dskip[c]);
            dbias[c] += ddt[c];
            if (a.z) {
              const float sg = sigmoid(zs[r][c]);
              dz[c] = dys[r][c] * fmaf(skip[c], xs[r][c], y[c]) * sg * fmaf(zs[r][c], 1.0f - sg, 1.0f);
            }
          }
          const int64_t at = ((int64_t)w.b * a.L + row_of(p, w.own, i)) * a.D + w.c0;
          store_n<T, 4, VEC>(static_cast<T*>(a.dx) + at, w.nc, dx);
          store_n<T, 4, VEC>(static_cast<T*>(a.ddt) + at, w.nc, ddt);
          if (a.dz) store_n<T, 4, VEC>(static_cast<T*>(a.dz) + at, w.nc, dz);
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (ENDS) {
    store_plane<G, NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, g);
    put_sums<SPLIT, G::CW>(sum, w.s, w.j, &s_dl[0][0]);
    __syncthreads();
    if (w.s == 0) {
      float v[4];
      get4(&s_dl[0][4 * w.j], v);
      store_n<float, 4, VEC>(p.chunk_s + ((int64_t)w.b * p.K + w.chunk) * a.D + w.c0, w.nc, v);
    }
    return;
  }
  if (a.dh0 && w.chunk == 0) store_dn<G, NS>(a.dh0 + (int64_t)w.b * a.D * a.N, a.N, w, g);
  store_plane<G, NS, VEC>(p.part_a + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, dA);
  put_sums<SPLIT, G::CW>(dskip, w.s, w.j, &s_1[0][0]);
  put_sums<SPLIT, G::CW>(dbias, w.s, w.j, &s_2[0][0]);
  __syncthreads();
  if (w.s == 0) {
    float u[4], v[4];
    get4(&s_1[0][4 * w.j], u);
    get4(&s_2[0][4 * w.j], v);
    float* to = p.part_d + ((int64_t)w.b * p.K + w.chunk) * 2 * a.D;
    store_n<float, 4, VEC>(to + w.c0, w.nc, u);
    store_n<float, 4, VEC>(to + a.D + w.c0, w.nc, v);
  }
}

// dB and dC: the waves' sums over their channels, added over a group's channel tiles in order, rounded once.
template <class T>
__global__ void __launch_bounds__(256) scan_bc_kernel(const ScanParams p, int NP) {
  const sed_scan_args& a = p.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rows = a.B * a.G * a.L;
  if (i >= rows * 2 * NP) return;
  const int e = (int)(i % (2 * NP)), n = e % NP;
  const int64_t r = i / (2 * NP), t = r % a.L, g = r / a.L % a.G, b = r / a.L / a.G;
  if (n >= a.N) return;
  const bool in = !a.frames || t < a.frames[b];
  float v = 0.0f;
  if (in) {
    const float* q = p.part_bc + ((b * a.G + g) * p.tiles * a.L + t) * (2 * NP) + e;
    for (int k = 0; k < p.tiles; ++k) v += q[(int64_t)k * a.L * 2 * NP];
  }
  static_cast<T*>(e < NP ? a.dB : a.dC)[((b * a.L + t) * a.G + g) * a.N + n] = (T)v;
}

// dA [D][N], d skip and d dt_bias [D]: sums over clips and chunks in order; dA's partial sums lie [NP][D].
__global__ void __launch_bounds__(256) scan_param_kernel(const ScanParams p, int NP) {
  const sed_scan_args& a = p.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)(a.N + 2) * a.D) return;
  const int64_t d = i % a.D, n = i / a.D, rows = a.B * p.K;
  const float* q = n < a.N ? p.part_a + n * a.D + d : p.part_d + (n - a.N) * a.D + d;
  const int64_t step = n < a.N ? (int64_t)NP * a.D : 2 * a.D;
  float v[4] = {0, 0, 0, 0};
  int64_t r = 0;
  for (; r + 4 <= rows; r += 4)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += q[(r + k) * step];
  for (; r < rows; ++r) v[0] += q[r * step];
  const float sum = (v[0] + v[1]) + (v[2] + v[3]);
  if (n < a.N)
    a.dA[d * a.N + n] = sum;
  else if (n == a.N) {
    if (a.dskip) a.dskip[d] = sum;
  } else if (a.ddt_bias)
    a.ddt_bias[d] = sum;
}

// ---- one frame ----------------------------------------------------------------------------------------------------------

// Bound: the states, read and written once.  A thread holds Q states of one channel (Q = 4: one 16-byte access), the
// SP = ceil(N / Q) threads of a channel are neighbours and each forms delta for itself.
template <class T, int Q, int SP>
__global__ void __launch_bounds__(256) scan_step_kernel(const sed_scan_args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int s = (int)(i % SP);
  const int64_t bd = i / SP;
  const bool in = bd < a.B * a.D;
  const int64_t d = in ? bd % a.D : 0, b = in ? bd / a.D : 0, g = d / (a.D / a.G);
  const float x = (float)static_cast<const T*>(a.x)[b * a.x_b + d];
  float v = (float)static_cast<const T*>(a.dt)[b * a.dt_b + d];
  if (a.dt_bias) v += a.dt_bias[d];
  const float dl = a.softplus ? softplus(v) : v, dx = dl * x;
  const T* Bp = static_cast<const T*>(a.Bm) + b * a.Bm_b + g * a.Bm_g;
  const T* Cp = static_cast<const T*>(a.Cm) + b * a.Cm_b + g * a.Cm_g;
  float* hp = a.h_last + (b * a.D + d) * a.N;
  float y = 0.0f;
  if (in) {
    if constexpr (Q == 4) {
      const int n0 = 4 * s;
      if (n0 < a.N) {
        f32x4 h = *reinterpret_cast<f32x4*>(hp + n0);
        const f32x4 A = *reinterpret_cast<const f32x4*>(a.A + d * a.N + n0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[k] = fmaf(exp2_hw(dl * kLog2e * A[k]), h[k], dx * (float)Bp[n0 + k]);
          y = fmaf((float)Cp[n0 + k], h[k], y);
        }
        *reinterpret_cast<f32x4*>(hp + n0) = h;
      }
    } else {
      for (int n = s; n < a.N; n += SP) {
        const float h = fmaf(exp2_hw(dl * kLog2e * a.A[d * a.N + n]), hp[n], dx * (float)Bp[n]);
        y = fmaf((float)Cp[n], h, y);
        hp[n] = h;
      }
    }
  }
  if (SP >= 2) y += dpp<kXor1>(y);
  if (SP >= 4) y += dpp<kXor2>(y);
  if (SP >= 8) y += dpp<kHalfMirror>(y);
  if (in && s == 0) {
    if (a.skip) y = fmaf(a.skip[d], x, y);
    if (a.z) {
      const float z = (float)static_cast<const T*>(a.z)[b * a.z_b + d];
      y *= z * sigmoid(z);
    }
    static_cast<T*>(a.y)[b * a.D + d] = (T)y;
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// Instance of a state count: NS states a lane, SPLIT lanes a channel.
struct Shape { int NS, SPLIT, NP, CW, TT; };
Shape shape_of(int N) {
  if (N <= 1) return {1, 1, 1, 256, 8};
  if (N <= 4) return {4, 1, 4, 256, 8};
  if (N <= 8) return {4, 2, 8, 128, 8};
  if (N <= 16) return {4, 4, 16, 64, 8};
  return {8, 4, 32, 64, 4};
}

struct Layout {
  int64_t L_chunk, saved_n;
  int32_t K, tiles;
  int64_t h, s, bc, pa, pd, total;  // float offsets into the workspace
};

// Chunks: 2048 waves keep the 1024 vector units busy; a chunk costs its frames almost twice (once for its end state, once for
// its outputs), so a clip stays whole where there are waves enough, and no chunk is shorter than two tiles.
Layout layout_of(const sed_scan_args& a, bool back) {
  const Shape s = shape_of(a.N);
  Layout l{};
  const int64_t cg = a.D / a.G;
  l.tiles = (int32_t)((cg + s.CW - 1) / s.CW);
  l.saved_n = (a.L + s.TT - 1) / s.TT;
  const int64_t waves = a.B * a.G * l.tiles, most = std::max<int64_t>(1, a.L / (2 * s.TT));
  int64_t K = waves >= 1024 ? 1 : std::min<int64_t>(most, (2048 + waves - 1) / waves);
  l.L_chunk = ((a.L + K - 1) / K + s.TT - 1) / s.TT * s.TT;
  K = std::max<int64_t>(1, (a.L + l.L_chunk - 1) / l.L_chunk);
  l.K = (int32_t)K;
  int64_t at = 0;
  const auto take = [&](int64_t n) { const int64_t o = at; at += (n + 63) / 64 * 64; return o; };
  if (K > 1) {
    l.h = take(a.B * K * s.NP * a.D);
    l.s = take(a.B * K * a.D);
  }
  if (back) {
    l.bc = take(a.B * a.G * l.tiles * a.L * 2 * s.NP);
    l.pa = take(a.B * K * s.NP * a.D);
    l.pd = take(a.B * K * 2 * a.D);
  }
  l.total = at;
  return l;
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_args(const sed_scan_args* a) {
  if (!a || a->B < 0 || a->L < 0 || a->D < 1 || a->N < 1 || a->N > 32 || a->G < 1 || a->D % a->G) return SED_ERR_BAD_ARG;
  if (a->dtype != SED_F32 && a->dtype != SED_BF16 && a->dtype != SED_F16) return SED_ERR_BAD_ARG;
  if (a->B > 0 && a->L > 0 && (!a->x || !a->dt || !a->A || !a->Bm || !a->Cm)) return SED_ERR_BAD_ARG;
  return SED_OK;
}

// Rows can be read 4 channels at a time.
bool vector_rows(const sed_scan_args& a, bool back) {
  const int64_t e = a.dtype == SED_F32 ? 4 : 2, bytes = 4 * e;
  const auto ok = [&](const void* p, int64_t sb, int64_t st) { return !p || (aligned(p, bytes) && sb % 4 == 0 && st % 4 == 0); };
  if (a.D / a.G % 4) return false;
  if (!ok(a.x, a.x_b, a.x_t) || !ok(a.dt, a.dt_b, a.dt_t) || !ok(a.z, a.z_b, a.z_t) || !aligned(a.saved, 16)) return false;
  if (!back) return aligned(a.y, bytes);
  return ok(a.dy, a.dy_b, a.dy_t) && aligned(a.dx, bytes) && aligned(a.ddt, bytes) && aligned(a.dz, bytes);
}

template <int NS, int SPLIT, class T, bool VEC>
int launch(const ScanParams& p, bool back, hipStream_t stream) {
  using G = Geo<NS, SPLIT>;
  const sed_scan_args& a = p.a;
  const int64_t grid = a.B * p.K * a.G * p.tiles, joins = (a.B * G::NP * a.D + 255) / 256;
  if (grid > 0x7fffffff || joins > 0x7fffffff) return SED_ERR_CAPACITY;
  if (!back) {
    if (p.K > 1) {
      scan_forward_kernel<NS, SPLIT, T, VEC, true><<<(unsigned)grid, 64, 0, stream>>>(p);
      chunk_join_kernel<false><<<(unsigned)joins, 256, 0, stream>>>(p, G::NP);
    }
    scan_forward_kernel<NS, SPLIT, T, VEC, false><<<(unsigned)grid, 64, 0, stream>>>(p);
    return seq_status(hipGetLastError());
  }
  const int64_t bc = (a.B * a.G * a.L * 2 * G::NP + 255) / 256, pr = ((a.N + 2) * a.D + 255) / 256;
  if (bc > 0x7fffffff) return SED_ERR_CAPACITY;
  if (p.K > 1) {
    scan_backward_kernel<NS, SPLIT, T, VEC, true><<<(unsigned)grid, 64, 0, stream>>>(p);
    chunk_join_kernel<true><<<(unsigned)joins, 256, 0, stream>>>(p, G::NP);
  }
  scan_backward_kernel<NS, SPLIT, T, VEC, false><<<(unsigned)grid, 64, 0, stream>>>(p);
  scan_bc_kernel<T><<<(unsigned)bc, 256, 0, stream>>>(p, G::NP);
  scan_param_kernel<<<(unsigned)pr, 256, 0, stream>>>(p, G::NP);
  return seq_status(hipGetLastError());
}

template <int NS, int SPLIT, class T>
int launch_v(const ScanParams& p, bool back, bool vec, hipStream_t s) {
  return vec ? launch<NS, SPLIT, T, true>(p, back, s) : launch<NS, SPLIT, T, false>(p, back, s);
}
template <int NS, int SPLIT>
int launch_t(const ScanParams& p, bool back, bool vec, hipStream_t s) {
  if (p.a.dtype == SED_F32) return launch_v<NS, SPLIT, float>(p, back, vec, s);
  if (p.a.dtype == SED_BF16) return launch_v<NS, SPLIT, bf16>(p, back, vec, s);
  return launch_v<NS, SPLIT, f16>(p, back, vec, s);
}

int run(const sed_scan_args* args, bool back, void* stream) {
  ScanParams p{};
  p.a = *args;
  const Layout l = layout_of(p.a, back);
  if (l.total > 0 && (!args->ws || args->ws_bytes < l.total * 4 || !aligned(args->ws, 16))) return SED_ERR_CAPACITY;
  float* ws = static_cast<float*>(args->ws);
  p.L_chunk = l.L_chunk;
  p.K = l.K;
  p.tiles = l.tiles;
  p.saved_n = (int32_t)l.saved_n;
  p.chunk_h = ws + l.h;
  p.chunk_s = ws + l.s;
  p.part_bc = ws + l.bc;
  p.part_a = ws + l.pa;
  p.part_d = ws + l.pd;
  const bool vec = vector_rows(p.a, back);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Shape sh = shape_of(p.a.N);
  if (sh.NP == 1) return launch_t<1, 1>(p, back, vec, s);
  if (sh.NP == 4) return launch_t<4, 1>(p, back, vec, s);
  if (sh.NP == 8) return launch_t<4, 2>(p, back, vec, s);
  if (sh.NP == 16) return launch_t<4, 4>(p, back, vec, s);
  return launch_t<8, 4>(p, back, vec, s);
}

template <class T>
int step(const sed_scan_args& a, hipStream_t s) {
  const bool four = a.N % 4 == 0 && aligned(a.h_last, 16) && aligned(a.A, 16);
  const int need = four ? a.N / 4 : a.N, SP = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
  const int64_t grid = (a.B * a.D * SP + 255) / 256;
  if (grid > 0x7fffffff) return SED_ERR_CAPACITY;
  const unsigned n = (unsigned)grid;
#define SED_STEP(Q, S) scan_step_kernel<T, Q, S><<<n, 256, 0, s>>>(a)
  if (four) {
    if (SP == 1) SED_STEP(4, 1);
    else if (SP == 2) SED_STEP(4, 2);
    else if (SP == 4) SED_STEP(4, 4);
    else SED_STEP(4, 8);
  } else {
    if (SP == 1) SED_STEP(1, 1);
    else if (SP == 2) SED_STEP(1, 2);
    else if (SP == 4) SED_STEP(1, 4);
    else SED_STEP(1, 8);
  }
#undef SED_STEP
  return seq_status(hipGetLastError());
}

}  // namespace
}  // namespace sed

extern "C" int64_t sed_gated_scan_saved_floats(int64_t B, int64_t L, int64_t D, int32_t N) {
  if (B < 0 || L < 0 || D < 1 || N < 1 || N > 32) return SED_ERR_BAD_ARG;
  const sed::Shape s = sed::shape_of(N);
  return B * ((L + s.TT - 1) / s.TT) * s.NP * D;
}

extern "C" int64_t sed_gated_scan_workspace(int64_t B, int64_t L, int64_t D, int32_t N, int32_t G, int32_t backward) {
  sed_scan_args a{};
  a.B = B, a.L = L, a.D = D, a.N = N, a.G = G;
  if (B < 0 || L < 0 || D < 1 || N < 1 || N > 32 || G < 1 || D % G) return SED_ERR_BAD_ARG;
  return sed::layout_of(a, backward != 0).total * 4;
}

extern "C" int sed_gated_scan_forward(const sed_scan_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->y) return SED_ERR_BAD_ARG;
  return sed::run(args, false, stream);
}

extern "C" int sed_gated_scan_backward(const sed_scan_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->dy || !args->saved || !args->dx || !args->ddt || !args->dB || !args->dC || !args->dA || (args->z && !args->dz)) return SED_ERR_BAD_ARG;
  return sed::run(args, true, stream);
}

extern "C" int sed_gated_scan_step(const sed_scan_args* args, void* stream) {
  const int rc = sed::check_args(args);
  if (rc != SED_OK) return rc;
  if (args->B == 0 || args->L == 0) return SED_OK;
  if (!args->h_last || !args->y || args->L != 1) return SED_ERR_BAD_ARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (args->dtype == SED_F32) return sed::step<float>(*args, s);
  if (args->dtype == SED_BF16) return sed::step<sed::bf16>(*args, s);
  return sed::step<sed::f16>(*args, s);
}
