// Gated linear recurrence along the frames of a clip, its gradient and its one-frame form, for gfx950.
//
//   delta_t[d] = softplus(dt_t[d] + dt_bias[d])   (or dt + dt_bias)
//   h_t[d,n]   = exp(delta_t[d] A[d,n]) h_{t-1}[d,n] + delta_t[d] x_t[d] B_t[g,n]
//   y_t[d]     = (sum_n C_t[g,n] h_t[d,n] + skip[d] x_t[d]) * silu(z_t[d])
//
// Bound: the vector unit.  A state takes one exp2 (two issue slots) and four multiply-adds per frame, and no matrix instruction
// helps, since the decay differs per channel, state and frame.  So the layout serves the vector unit: a wave works by itself,
// every lane holds 4 channels x NS states in registers and walks along the frames, SPLIT lanes share a channel's NP = NS * SPLIT
// states.  B and C are then read from LDS once for 4 channels, the sum over states is NS multiply-adds and a few lane exchanges
// for 4 channels at once, and in the gradient the sum over channels is 4 multiply-adds in the lane before any exchange.
// Frames come in tiles of TT rows: the lanes load a tile's rows (each row once), form delta and delta * x in LDS, scan, and
// write the finished rows, while the next tile's rows are on their way.
//
// A clip is cut into chunks where there are too few waves to fill the card: a first pass gives every chunk's own end state
// from zero and the sum of its delta (the decay over a chunk is exp(A * sum), no product of decays is kept), the ends are joined
// in order, and the main pass starts each chunk from its state.  The gradient is the same recurrence from the other end:
// g_t = C_t gy_t + exp(delta_{t+1} A) g_{t+1}.  It recomputes a tile's states from the state in front of the tile, which the
// forward pass keeps (`saved`), and keeps exp(delta A) h_{t-1} of TB frames in registers; keeping the decays as well, or all of a
// tile's frames, was slower for the registers it took (two waves a unit need 256 at most).
// States, decays and sums are fp32; x, dt, z, B, C, y and their gradients are fp32, bf16 or fp16, rounded once at the store.
//
// Measured (MI355X, bf16, N = 16): 16 x 513 x 1536 forward 107 us in one pass of thin waves (46 + 67 in chunks of wide ones), 1.9e12
// states of a frame a second; its gradient 190 .. 203 us and 50 .. 53 us for the chunks' ends: 26.5 vector instructions a state and
// frame, of which 16 are the formulas', the vector units issuing 76 % of the time.  64 clips of up to 1024 x 768, 31759 frames
// together: 169 us.
// 512 streams x 1536 x 16, one frame: 25 us for 107 MB (4.2 TB/s; a 1 GiB copy reaches 5.1).
#include "seq_core.h"

#include <algorithm>

namespace sed {
namespace {

struct ScanParams {
  sed_scan_args a;
  int32_t ns;       // states kept of a clip, ceil(L / TS)
  int32_t four;     // N % 4 == 0 and A, h0, dh_last are aligned to 16 bytes
  int32_t K;        // chunks of a clip
  int32_t tiles;    // channel tiles of a group
  float* chunk_h;   // [B][K][NP][D]  end states from zero, then the states in front of the chunks
  float* chunk_s;   // [B][K][D]      half the sums of delta
  float* part_bc;   // [B][G * tiles][L][2 * NP]  dB, dC of one wave's channels
  float* part_a;    // [B * K][D * NP] dA  [NP][D] per row
  float* part_d;    // [B * K][2][D]  d skip, d dt_bias
};

// Up to this many chunks every chunk forms the state in front of it from the ends of the others by itself, which is little work
// and saves a launch; beyond, chunk_join_kernel does it once for all.
constexpr int kOwnJoin = 32;

// Waves of a workgroup.  They work apart from each other (own LDS, no barrier): one workgroup to start for four of them (the
// forward pass over 16 x 513 x 1536 x 16 takes 113 us so, 121 with one).  The gradient's fp32 tiles take 21 KB of LDS a wave: by
// fours, only one workgroup would fit.
template <class T, bool BACK, bool ENDS>
constexpr int waves_of() { return BACK && !ENDS && sizeof(T) == 4 ? 1 : 4; }
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }
// What a wave's lanes wrote to LDS is there for its other lanes: a wave's LDS operations are carried out in order, so only the
// compiler has to keep to it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Tile geometry of one instance.
template <int NS, int SPLIT>
struct Geo {
  static constexpr int NP = NS * SPLIT;       // states, padded
  static constexpr int J = 64 / SPLIT;        // lanes along channels
  static constexpr int CW = 4 * J;            // channels of a wave
  static constexpr int TT = SPLIT == 16 ? 16 : SPLIT >= 4 ? 8 : 4;  // frames of a tile
  static constexpr int TS = NP >= 8 ? 8 : 4;  // frames from one kept state to the next, whatever the tile
  static constexpr int TB = 4;                // frames whose states the gradient holds at a time: 16 NS <= 64 registers
  static constexpr int R = TT / SPLIT;        // rows a lane loads
  static constexpr int PB = (TT * NP + 63) / 64;
  static_assert(R * SPLIT == TT, "");
};

// LDS that a wave of the main passes takes (the gradient keeps rows of elements of `size` bytes there), and its waves on a vector unit.
constexpr int lds_of(int NS, int SPLIT, int NP, int TT, bool back, int size) {
  const int cw = 256 / SPLIT;
  if (!back) return 4 * (3 * TT * cw + 2 * TT * NP);
  return 4 * (4 * TT * cw + 2 * TT * NP + NS * 256 + 2 * cw) + 4 * (TT / SPLIT) * 64 * 4 * size;
}
constexpr int per_unit(int SPLIT, bool back) { return back ? 2 : SPLIT == 1 ? 3 : 4; }

// Where a wave works.
struct Where {
  int b, chunk, g, s, j;
  int own;         // frames of the clip's own
  int begin, end;  // the chunk's frames of the clip's own
  int c0, cl;      // first channel of the lane; the same, or the group's first where the lane has none
  int nc;          // channels of the lane (0..4)
  int tile;        // over all groups
  int flip;        // TT - 1 where the walk goes to earlier rows
};

// First frame of a clip's chunk k < K: its own tiles in K even parts, so that clips of other lengths have other chunks, but none
// begins behind the clip's own frames (a clip of fewer than K tiles has empty ones).  Behind the last one: the end.
template <class G>
__device__ __forceinline__ int chunk_begin(const ScanParams& p, int own, int k) {
  return std::min((int)((int64_t)k * ((own + G::TT - 1) / G::TT) / p.K) * G::TT, own);
}

// The clip that place q of the batch stands for.  Clips of other lengths are started by 64, the longest ones first, so that the last
// waves to end are short ones: 64 clips of up to 1024 x 768 x 16 (31759 frames together, the longest 1009) forward take 169 us, 223 in the
// batch's own order; both passes of another batch's gradient 563 us, 634.  A wave ranks its 64 clips by itself, 5 instructions each.
__device__ __forceinline__ int by_length(const sed_scan_args& a, int q) {
  const int lane = threadIdx.x % 64, first = q & ~63, n = (int)std::min<int64_t>(64, a.B - first);
  const int mine = lane < n ? std::max(0, std::min((int)a.L, a.frames[first + lane])) : -1;
  int longer = 0;
  for (int j = 0; j < n; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    longer += other > mine || (other == mine && j < lane);
  }
  return first + __builtin_ctzll(__ballot(longer == q - first));
}

template <class G, int WAVES>
__device__ __forceinline__ Where where(const ScanParams& p) {
  Where w;
  const sed_scan_args& a = p.a;
  const unsigned all = p.tiles * a.G;
  unsigned i = blockIdx.x * WAVES + wave_id();
  w.tile = i % all;
  i /= all;
  w.chunk = i % p.K;
  w.b = i / p.K;  // B or more in the last workgroup's spare waves, which leave at once
  if (a.frames && w.b < a.B) w.b = by_length(a, w.b);
  w.g = w.tile / p.tiles;
  w.flip = a.reverse ? G::TT - 1 : 0;
  w.s = threadIdx.x % 64 / G::J;
  w.j = threadIdx.x % G::J;
  const int cg = (int)a.D / a.G, in = (w.tile % p.tiles) * G::CW + 4 * w.j;
  w.c0 = w.g * cg + in;
  w.nc = std::max(0, std::min(4, cg - in));
  w.cl = w.nc ? w.c0 : w.g * cg;
  w.own = (int)a.L;
  if (a.frames) w.own = std::max(0, std::min((int)a.L, a.frames[std::min<int64_t>(w.b, a.B - 1)]));
  w.begin = chunk_begin<G>(p, w.own, w.chunk);
  w.end = chunk_begin<G>(p, w.own, w.chunk + 1);
  return w;
}

// Row of the clip that comes i-th: behind the clip's own rows every row is itself.
__device__ __forceinline__ int row_of(const ScanParams& p, int own, int i) { return p.a.reverse && i < own ? own - 1 - i : i; }

template <class T>
using T4 = T __attribute__((ext_vector_type(4)));

// Rows of a tensor in the order of the walk.  An address is a uniform base that moves with the tile (a scalar) and 32 bits of
// the lane's own: row i0 + t lies t rows behind the tile's first, or TT - 1 - t = t ^ (TT - 1) behind the tile's last where the
// walk goes to earlier rows, so the lane's part is never negative.  Rows are at most 2^26 elements apart (checked on the host).
template <class G, class T>
struct Rows {
  const char* base;  // tile of i0 = 0
  int32_t step;      // bytes from one frame of the walk to the next
  __device__ __forceinline__ Rows(const ScanParams& q, const Where& w, const void* p, int64_t sb, int64_t st) {
    const int64_t bytes = st * (int64_t)sizeof(T);
    step = (int32_t)(q.a.reverse ? -bytes : bytes);
    base = static_cast<const char*>(p) + w.b * sb * (int64_t)sizeof(T) + (q.a.reverse ? (int64_t)(w.own - G::TT) * bytes : 0);
  }
  __device__ __forceinline__ const char* tile(int i0) const { return base + (int64_t)i0 * step; }
  __device__ __forceinline__ uint32_t lane(const Where& w, uint32_t t, uint32_t c) const { return (t ^ w.flip) * (uint32_t)(w.flip ? -step : step) + c * (uint32_t)sizeof(T); }
};

// 4 channels of the rows i0 + r * SPLIT + s of a tile.  Every load is in bounds, so none is conditional: rows behind the clip's
// own read its last one, lanes and channels without a channel read one that exists; what they read is replaced where it is used.
template <class G, class T, bool VEC>
__device__ __forceinline__ void load_rows(const Rows<G, T>& rows, const Where& w, int i0, T4<T> (&out)[G::R]) {
  const char* at = rows.tile(i0);
#pragma unroll
  for (int r = 0; r < G::R; ++r) {
    const T* q = reinterpret_cast<const T*>(at + rows.lane(w, std::min(r * (64 / G::J) + w.s, w.own - 1 - i0), w.cl));
    if constexpr (VEC) {
      out[r] = *reinterpret_cast<const T4<T>*>(q);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) out[r][c] = q[c < w.nc ? c : 0];
    }
  }
}

// One of the same rows of an output; rows behind the clip's own are not written.
template <class G, class T, bool VEC>
__device__ __forceinline__ void store_row(const Rows<G, T>& rows, const Where& w, int i0, int r, const float (&v)[4]) {
  const int t = r * (64 / G::J) + w.s;
  store_n<T, 4, VEC>(reinterpret_cast<T*>(const_cast<char*>(rows.tile(i0)) + rows.lane(w, t, w.c0)), i0 + t < w.own ? w.nc : 0, v);
}

// B or C of a tile: element e = lane + 64 k is state e % NP of row e / NP.
template <class G, class T>
__device__ __forceinline__ void load_states(const Rows<G, T>& rows, const ScanParams& q, const Where& w, int i0, T (&out)[G::PB]) {
  const char* at = rows.tile(i0);
  const int last = std::min(w.own - 1 - i0, G::TT - 1);
#pragma unroll
  for (int k = 0; k < G::PB; ++k) {
    const int e = w.s * G::J + w.j + 64 * k, n = e % G::NP, t = e / G::NP;
    out[k] = *reinterpret_cast<const T*>(at + rows.lane(w, std::min(t, last), n < q.a.N ? n : 0));
  }
}
// Into LDS; the padding states are zero, and so are rows behind the clip's own.
template <class G, class T>
__device__ __forceinline__ void put_states(const ScanParams& q, const Where& w, int i0, const T (&v)[G::PB], float* to) {
#pragma unroll
  for (int k = 0; k < G::PB; ++k) {
    const int e = w.s * G::J + w.j + 64 * k, n = e % G::NP, t = e / G::NP;
    if (G::TT * G::NP % 64 == 0 || e < G::TT * G::NP) to[e] = n < q.a.N && i0 + t < w.own ? (float)v[k] : 0.0f;
  }
}

template <int NS>
__device__ __forceinline__ void get_states(const float* from, float (&v)[NS]) {
  if constexpr (NS == 4) {
    const f32x4 t = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = t[i];
  } else if constexpr (NS == 2) {
    const f32x2 t = *reinterpret_cast<const f32x2*>(from);
    v[0] = t[0];
    v[1] = t[1];
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

// What a frame of a tile needs out of LDS; row, state: the lane's places in the tile's first frame.
template <int NS>
struct Step {
  float dl[4], dx[4], gy[4], B[NS], C[NS];
  template <class G, bool X, bool GY, bool WITH_C>
  __device__ __forceinline__ void get(int row, int state, int t, const float* s_dl, const float* s_dx, const float* s_gy, const float* s_B, const float* s_C) {
    get4(s_dl + row + t * G::CW, dl);
    if (X) get4(s_dx + row + t * G::CW, dx);
    if (X) get_states<NS>(s_B + state + t * G::NP, B);
    if (GY) get4(s_gy + row + t * G::CW, gy);
    if (WITH_C) get_states<NS>(s_C + state + t * G::NP, C);
  }
};

// Writes the sums of v[4] over the SPLIT lanes that share a channel to the lane group's 4 places.
template <int SPLIT>
__device__ __forceinline__ void put_sums(const float (&v)[4], int s, float* at) {
  if constexpr (SPLIT >= 4) {
    // rows of 16 lanes: halves of the wave first (channels 0 | 2 and 1 | 3), then neighbouring rows; with SPLIT = 8 and 16 two
    // and four groups of lanes in a row hold the same channel
    float u = fold16(fold32(v[0], v[2]), fold32(v[1], v[3]));
    if (SPLIT >= 8) u += dpp<kRor8>(u);
    if (SPLIT >= 16) u += dpp<kRor4>(u);
    at[s / (SPLIT / 4)] = u;
  } else if constexpr (SPLIT == 2) {
    *reinterpret_cast<f32x2*>(at + 2 * s) = f32x2{fold32(v[0], v[2]), fold32(v[1], v[3])};
  } else {
    put4(v, at);
  }
}

template <bool VEC = false>
__device__ __forceinline__ void per_channel(const float* from, const Where& w, float (&v)[4]) {
  if constexpr (VEC) {
    get4(from + w.cl, v);
    return;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = from ? from[w.cl + (c < w.nc ? c : 0)] : 0.0f;
}

// states of a lane from / to a [NP][D] plane: a uniform base per state and 32 bits of the lane's own (32 D floats at most)
template <int NS, bool VEC>
__device__ __forceinline__ void load_plane(const float* plane, int64_t D, const Where& w, float (&h)[4][NS]) {
  const uint32_t off = (uint32_t)(w.s * NS * (int)D + w.cl) * 4u;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const float* q = reinterpret_cast<const float*>(reinterpret_cast<const char*>(plane + n * D) + off);
    if constexpr (VEC) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(q);
#pragma unroll
      for (int c = 0; c < 4; ++c) h[c][n] = v[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) h[c][n] = q[c < w.nc ? c : 0];
    }
  }
}
template <int NS, bool VEC>
__device__ __forceinline__ void store_plane(float* plane, int64_t D, const Where& w, const float (&h)[4][NS]) {
  const uint32_t off = (uint32_t)(w.s * NS * (int)D + w.c0) * 4u;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = h[c][n];
    store_n<float, 4, VEC>(reinterpret_cast<float*>(reinterpret_cast<char*>(plane + n * D) + off), w.nc, v);
  }
}
// states of a lane from / to the caller's [D][N]; padding states are zero, a lane without a channel reads another's
template <int NS>
__device__ __forceinline__ void load_dn(const ScanParams& p, const float* base, const Where& w, float (&h)[4][NS]) {
  const int N = p.a.N;
  if (NS == 4 && p.four) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(base + (int64_t)(w.cl + (c < w.nc ? c : 0)) * N + std::min(w.s * NS, N - 4));
#pragma unroll
      for (int n = 0; n < NS; ++n) h[c][n] = w.s * NS < N ? v[n % 4] : 0.0f;
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int k = w.s * NS + n;
      const float v = base[(int64_t)(w.cl + (c < w.nc ? c : 0)) * N + std::min(k, N - 1)];
      h[c][n] = k < N ? v : 0.0f;
    }
}
// A in units of exp2.  Its lowest values stay finite, so that a step of zero (a lane without a channel, a frame behind the clip's own, a
// chunk without frames) keeps its state: 0 times infinity would be a NaN.
__device__ __forceinline__ float exponent(float A) {
  const float v = A * kLog2e;
  return __builtin_amdgcn_classf(v, 4) ? -3.4028235e38f : v;  // -infinity
}
template <int NS>
__device__ __forceinline__ void load_exponents(const ScanParams& p, const Where& w, float (&A2)[4][NS]) {
  load_dn<NS>(p, p.a.A, w, A2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) A2[c][n] = exponent(A2[c][n]);
}
template <int NS>
__device__ __forceinline__ void store_dn(float* base, int N, const Where& w, const float (&h)[4][NS]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int k = w.s * NS + n;
      if (c < w.nc && k < N) base[(int64_t)(w.c0 + c) * N + k] = h[c][n];
    }
}

// delta of a tile's rows; zero where the row or the channel is none (exp(0) = 1 leaves the state as it is)
template <class G, class T, bool VEC>
__device__ __forceinline__ void deltas(const ScanParams& p, const Where& w, int i0, const T4<T> (&dt)[G::R], const float (&bias)[4], float (&dl)[G::R][4]) {
#pragma unroll
  for (int r = 0; r < G::R; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) dl[r][c] = (float)dt[r][c] + bias[c];
  if (p.a.softplus) {
#pragma unroll
    for (int r = 0; r < G::R; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) dl[r][c] = softplus(dl[r][c]);
  }
#pragma unroll
  for (int r = 0; r < G::R; ++r) {
    const bool in = i0 + r * (64 / G::J) + w.s < w.own;
#pragma unroll
    for (int c = 0; c < 4; ++c) dl[r][c] = in && (VEC ? w.nc > 0 : c < w.nc) ? dl[r][c] : 0.0f;
  }
}
// v where the row and the channel exist (a row behind the clip's own can hold anything)
template <class G, bool VEC>
__device__ __forceinline__ void only_own(const Where& w, int i0, int r, float (&v)[4]) {
  const bool in = i0 + r * (64 / G::J) + w.s < w.own;
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = in && (VEC ? w.nc > 0 : c < w.nc) ? v[c] : 0.0f;
}

// 4^z h + e over a chunk, z half the sum of its frames' exponents.  In two steps, the second to the scaled state: the frames one by one
// carry a state of zero, or a small one, through growth that is beyond fp32 as a whole (A delta > 0), and so does this (0 times
// infinity would be a NaN).  A NaN in z is in e as well.
__device__ __forceinline__ float pass_chunk(float z, float h, float e) {
  const float f = exp2_hw(fminf(z, 127.0f));
  return fmaf(f, f * h, e);
}

// The state behind `count` chunks from the state h in front of them (their end states from zero and sums of delta, halved): chunks
// q, q + step, ..  A chunk's values are on their way while the one in front of it is worked on.
template <class G, int NS, bool VEC>
__device__ __forceinline__ void pass_chunks(const ScanParams& p, const Where& w, int q, int step, int count, const float (&A2)[4][NS], float (&h)[4][NS]) {
  if (count <= 0) return;
  const int64_t D = p.a.D;
  float e[4][NS], s[4];
  const auto load = [&](int i) {
    const int64_t at = (int64_t)w.b * p.K + q + i * step;
    load_plane<NS, VEC>(p.chunk_h + at * G::NP * D, D, w, e);
    per_channel<VEC>(p.chunk_s + at * D, w, s);
  };
  load(0);
#pragma unroll 2
  for (int i = 0; i < count; ++i) {
    float e1[4][NS], s1[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s1[c] = s[c];
#pragma unroll
      for (int n = 0; n < NS; ++n) e1[c][n] = e[c][n];
    }
    if (i + 1 < count) load(i + 1);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int n = 0; n < NS; ++n) h[c][n] = pass_chunk(A2[c][n] * s1[c], h[c][n], e1[c][n]);
      __builtin_amdgcn_sched_barrier(0);  // all at once they would take the registers of the rows on their way
    }
  }
}

// Zero rows of the clip behind its own, this chunk's share of them.
template <class G, class T, bool VEC>
__device__ __forceinline__ void clear_rows(const ScanParams& p, const Where& w, void* base) {
  const float zero[4] = {0, 0, 0, 0};
  const int64_t behind = p.a.L - w.own;
  const int stop = w.own + (int)(behind * (w.chunk + 1) / p.K);
  for (int i = w.own + (int)(behind * w.chunk / p.K) + w.s; i < stop; i += 64 / G::J)
    store_n<T, 4, VEC>(static_cast<T*>(base) + ((int64_t)w.b * p.a.L + i) * p.a.D + w.c0, w.nc, zero);
}


// ---- forward ------------------------------------------------------------------------------------------------------------

// ENDS: only the chunk's end state from zero and its sum of delta.  Otherwise the chunk's outputs.
template <int NS, int SPLIT, class T, bool VEC, bool ENDS>
__global__ void __launch_bounds__((64 * waves_of<T, false, ENDS>()), (per_unit(SPLIT, false))) scan_forward_kernel(const ScanParams p) {
  using G = Geo<NS, SPLIT>;
  constexpr int W = waves_of<T, false, ENDS>();
  const sed_scan_args& a = p.a;
  const Where w = where<G, W>(p);
  struct Shared {
    float dl[G::TT][G::CW], dx[G::TT][G::CW], y[ENDS ? 1 : G::TT][G::CW], B[G::TT][G::NP], C[G::TT][G::NP];
  };
  static_assert(ENDS || sizeof(Shared) == lds_of(NS, SPLIT, G::NP, G::TT, false, sizeof(T)), "");
  __shared__ __attribute__((aligned(16))) Shared shared[W];
  Shared& sh = shared[wave_id()];
  auto &s_dl = sh.dl, &s_dx = sh.dx;
  auto &s_y = sh.y;
  auto &s_B = sh.B, &s_C = sh.C;
  if (w.b >= a.B) return;
  if (ENDS && (w.chunk == p.K - 1 || w.own == 0)) return;  // nothing comes behind it
  if (!ENDS) {
    clear_rows<G, T, VEC>(p, w, a.y);
    if (w.own == 0) {
      if (a.h_last && w.chunk == 0) {
        float h[4][NS] = {};
        if (a.h0) load_dn<NS>(p, a.h0 + (int64_t)w.b * a.D * a.N, w, h);
        store_dn<NS>(a.h_last + (int64_t)w.b * a.D * a.N, a.N, w, h);
      }
      return;
    }
  }

  const Rows<G, T> rx(p, w, a.x, a.x_b, a.x_t), rdt(p, w, a.dt, a.dt_b, a.dt_t), rz(p, w, a.z, a.z_b, a.z_t), ry(p, w, a.y, a.L * a.D, a.D);
  const Rows<G, T> rB(p, w, static_cast<const T*>(a.Bm) + w.g * a.Bm_g, a.Bm_b, a.Bm_t), rC(p, w, static_cast<const T*>(a.Cm) + w.g * a.Cm_g, a.Cm_b, a.Cm_t);
  T4<T> x[G::R], dt[G::R], z[G::R];
  T bv[G::PB], cv[G::PB];
  const auto fetch = [&](int i0) {
    load_rows<G, T, VEC>(rx, w, i0, x);
    load_rows<G, T, VEC>(rdt, w, i0, dt);
    load_states<G, T>(rB, p, w, i0, bv);
    if (!ENDS) {
      if (a.z) load_rows<G, T, VEC>(rz, w, i0, z);
      load_states<G, T>(rC, p, w, i0, cv);
    }
  };
  fetch(w.begin);

  float A2[4][NS], h[4][NS], bias[4], skip[4], sum[4] = {0, 0, 0, 0};
  load_exponents<NS>(p, w, A2);
  per_channel(a.dt_bias, w, bias);
  per_channel(a.skip, w, skip);
  if (!ENDS && p.K > kOwnJoin) {
    load_plane<NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, h);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < NS; ++n) h[c][n] = 0.0f;
    if (!ENDS && a.h0) load_dn<NS>(p, a.h0 + (int64_t)w.b * a.D * a.N, w, h);
    if (!ENDS) pass_chunks<G, NS, VEC>(p, w, 0, 1, w.chunk, A2, h);
  }

  for (int i0 = w.begin; i0 < w.end; i0 += G::TT) {
    T4<T> xs[G::R], zs[G::R];
    float dl[G::R][4];
    deltas<G, T, VEC>(p, w, i0, dt, bias, dl);
#pragma unroll
    for (int r = 0; r < G::R; ++r) {
      float dx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        dx[c] = dl[r][c] * (float)x[r][c];
        if (ENDS) sum[c] += dl[r][c];
      }
      only_own<G, VEC>(w, i0, r, dx);
      put4(dl[r], &s_dl[r * SPLIT + w.s][4 * w.j]);
      put4(dx, &s_dx[r * SPLIT + w.s][4 * w.j]);
      xs[r] = x[r];
      zs[r] = z[r];
    }
    put_states<G, T>(p, w, i0, bv, &s_B[0][0]);
    if (!ENDS) put_states<G, T>(p, w, i0, cv, &s_C[0][0]);
    if (i0 + G::TT < w.end) fetch(i0 + G::TT);
    wave_sync();
    // a frame's values are read while the frame in front of it is worked on
    const int row = 4 * w.j, state = w.s * NS;
    Step<NS> f[2];
    f[0].template get<G, true, false, !ENDS>(row, state, 0, s_dl[0], s_dx[0], nullptr, s_B[0], s_C[0]);
#pragma unroll
    for (int t = 0; t < G::TT; ++t) {
      const Step<NS>& q = f[t % 2];
      if (!ENDS && a.saved && t % G::TS == 0 && i0 + t < w.own)
        store_plane<NS, VEC>(a.saved + ((int64_t)w.b * p.ns + (i0 + t) / G::TS) * G::NP * a.D, a.D, w, h);
      if (t + 1 < G::TT) f[(t + 1) % 2].template get<G, true, false, !ENDS>(row, state, t + 1, s_dl[0], s_dx[0], nullptr, s_B[0], s_C[0]);
      float y[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        y[c] = 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          h[c][n] = fmaf(exp2_hw(q.dl[c] * A2[c][n]), h[c][n], q.dx[c] * q.B[n]);
          if (!ENDS) y[c] = fmaf(q.C[n], h[c][n], y[c]);
        }
      }
      if (!ENDS) put_sums<SPLIT>(y, w.s, &s_y[t][4 * w.j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wave_sync();
    if (!ENDS) {
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        float y[4];
        get4(&s_y[r * SPLIT + w.s][4 * w.j], y);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = fmaf(skip[c], (float)xs[r][c], y[c]);
        if (a.z) {
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] *= (float)zs[r][c] * sigmoid((float)zs[r][c]);
        }
        store_row<G, T, VEC>(ry, w, i0, r, y);
      }
      wave_sync();
    }
  }
  if (ENDS) {
    store_plane<NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, h);
    // every lane of a channel summed its own rows
    wave_sync();
    put_sums<SPLIT>(sum, w.s, &s_dl[0][4 * w.j]);
    wave_sync();
    if (w.s == 0) {
      float v[4];
      get4(&s_dl[0][4 * w.j], v);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] *= 0.5f;
      store_n<float, 4, VEC>(p.chunk_s + ((int64_t)w.b * p.K + w.chunk) * a.D + w.c0, w.nc, v);
    }
  } else if (a.h_last && w.chunk == p.K - 1) {
    store_dn<NS>(a.h_last + (int64_t)w.b * a.D * a.N, a.N, w, h);
  }
}

// The states in front of the chunks, over the chunks in order (BACK: the gradients behind them, from the last).
// In: every chunk's end state from zero; out, in its place: the state it starts from.  A block has 1024 / SEG (channel, state)
// pairs next to each other in memory and SEG lanes for each, which take a run of chunks: first the run's own end and sum, then
// the runs in order (LDS), then the run again from its start, so that a long clip's chunks are not one long chain of loads
// (1 x 100000 x 16 x 16 forward: 64 us with 16 lanes, 49 with 32, 45 with 64).
template <class G, bool BACK>
__global__ void __launch_bounds__(1024) chunk_join_kernel(const ScanParams p) {
  const sed_scan_args& a = p.a;
  constexpr int NP = G::NP, SEG = 64, W = 1024 / SEG;
  __shared__ float s_h[SEG][W], s_s[SEG][W];
  const int seg = threadIdx.x / W, lane = threadIdx.x % W;
  const int64_t i = (int64_t)blockIdx.x * W + lane;
  const bool live = i < a.B * NP * a.D;
  const int64_t d = live ? i % a.D : 0, n = live ? i / a.D % NP : 0, b = live ? i / a.D / NP : 0;
  int own = (int)a.L;
  if (a.frames) own = std::max(0, std::min((int)a.L, a.frames[b]));
  const int k_own = own > 0 ? p.K : 0;
  const bool real = n < a.N;
  const float A2 = real ? exponent(a.A[d * a.N + n]) : 0.0f;
  const float* first = BACK ? a.dh_last : a.h0;
  float* hp = p.chunk_h + (b * p.K * NP + n) * a.D + d;
  const float* sp = p.chunk_s + b * p.K * a.D + d;
  const int per = (k_own + SEG - 1) / SEG, q0 = seg * per, q1 = live ? std::min(q0 + per, k_own) : 0;
  const auto at = [&](int q) { return (int64_t)(BACK ? k_own - 1 - q : q); };
  // the last chunk of the walk hands nothing on
  {
    float h = 0.0f, s = 0.0f;
#pragma unroll 4
    for (int q = q0; q < std::min(q1, k_own - 1); ++q) {
      const float sk = sp[at(q) * a.D];
      h = pass_chunk(A2 * sk, h, hp[at(q) * NP * a.D]);
      s += sk;
    }
    s_h[seg][lane] = h;
    s_s[seg][lane] = s;
    __syncthreads();
  }
  float h = first && real && live ? first[(b * a.D + d) * a.N + n] : 0.0f;
  for (int k = 0; k < seg; ++k) h = pass_chunk(A2 * s_s[k][lane], h, s_h[k][lane]);
#pragma unroll 4
  for (int q = q0; q < q1; ++q) {
    const bool more = q < k_own - 1;
    const float end = more ? hp[at(q) * NP * a.D] : 0.0f, sk = more ? sp[at(q) * a.D] : 0.0f;
    hp[at(q) * NP * a.D] = h;
    h = pass_chunk(A2 * sk, h, end);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------

// Sums of NV values over the J lanes that share states: returned in lane j is the sum of v[sum_index(j)].
template <int NV, int J>
__device__ __forceinline__ float sum_lanes(float (&v)[NV], int j) {
  int n = NV;
#pragma unroll
  for (int bit = J / 2; bit >= 1; bit /= 2) {
    const auto other = [&](float x) {
      return bit == 8 ? dpp<kRor8>(x) : bit == 4 ? dpp<kHalfMirror>(x) : bit == 2 ? dpp<kXor2>(x) : dpp<kXor1>(x);
    };
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i)
        if (i < n) {
          if (bit == 32) v[i] = fold32(v[i], v[i + n]);
          if (bit == 16) v[i] = fold16(v[i], v[i + n]);
          if (bit < 16) {
            const float lo = v[i] + other(v[i]), hi = v[i + n] + other(v[i + n]);
            v[i] = j & bit ? hi : lo;
          }
        }
    } else {
      v[0] = bit == 32 ? fold32(v[0], v[0]) : bit == 16 ? fold16(v[0], v[0]) : v[0] + other(v[0]);
    }
  }
  return v[0];
}
// The value lane j holds, or -1 where a lane in front of it holds the same.
template <int NV, int J>
__device__ __forceinline__ int sum_index(int j) {
  int n = NV, index = 0;
  bool first = true;
#pragma unroll
  for (int bit = J / 2; bit >= 1; bit /= 2) {
    if (n > 1) {
      n /= 2;
      if (j & bit) index += n;
    } else if (j & bit) {
      first = false;
    }
  }
  return first ? index : -1;
}

// ENDS: only the gradient that reaches the frame in front of the chunk from the chunk's own outputs, and the sum of delta.
template <int NS, int SPLIT, class T, bool VEC, bool ENDS>
__global__ void __launch_bounds__((64 * waves_of<T, true, ENDS>()), (ENDS ? 4 : per_unit(SPLIT, true))) scan_backward_kernel(const ScanParams p) {
  using G = Geo<NS, SPLIT>;
  constexpr int W = waves_of<T, true, ENDS>();
  const sed_scan_args& a = p.a;
  Where w = where<G, W>(p);
  constexpr int TX = ENDS ? 1 : G::TT, TB = G::TB;
  constexpr bool EARLY = NS <= 2;  // dC is summed while the states are formed: a multiply-add less, TB * NS registers more
  // a row's gy and dx make room for the sums S2 and S1 that its frame leaves behind; raw, h: the tile's rows and the state in
  // front of it, each lane its own (registers are short); ch: dt_bias and skip
  struct Shared {
    float dl[G::TT][G::CW], gy[G::TT][G::CW], dx[TX][G::CW], y[TX][G::CW], B[G::TT][G::NP], C[G::TT][G::NP];
    T4<T> raw[ENDS ? 1 : 4][ENDS ? 1 : G::R][64];
    float h[ENDS ? 1 : NS][ENDS ? 4 : 256], ch[2][G::CW];
  };
  static_assert(ENDS || sizeof(Shared) == lds_of(NS, SPLIT, G::NP, G::TT, true, sizeof(T)), "");
  __shared__ __attribute__((aligned(16))) Shared shared[W];
  Shared& sh = shared[wave_id()];
  auto &s_dl = sh.dl, &s_gy = sh.gy;
  auto &s_dx = sh.dx, &s_y = sh.y;
  auto &s_B = sh.B, &s_C = sh.C;
  auto& s_raw = sh.raw;
  auto& s_h = sh.h;
  auto& s_ch = sh.ch;
  if (w.b >= a.B) return;
  float(&s_1)[TX][G::CW] = s_dx;
  if (ENDS && (w.chunk == 0 || w.own == 0)) return;

  // rows behind the clip's own have no gradient
  if (!ENDS) {
    clear_rows<G, T, VEC>(p, w, a.dx);
    clear_rows<G, T, VEC>(p, w, a.ddt);
    if (a.dz) clear_rows<G, T, VEC>(p, w, a.dz);
  }
  const int tiles = w.begin < w.end ? (w.end - w.begin + G::TT - 1) / G::TT : 0;

  const Rows<G, T> rx(p, w, a.x, a.x_b, a.x_t), rdt(p, w, a.dt, a.dt_b, a.dt_t), rz(p, w, a.z, a.z_b, a.z_t), rdy(p, w, a.dy, a.dy_b, a.dy_t);
  const Rows<G, T> rB(p, w, static_cast<const T*>(a.Bm) + w.g * a.Bm_g, a.Bm_b, a.Bm_t), rC(p, w, static_cast<const T*>(a.Cm) + w.g * a.Cm_g, a.Cm_b, a.Cm_t);
  const Rows<G, T> wx(p, w, a.dx, a.L * a.D, a.D), wdt(p, w, a.ddt, a.L * a.D, a.D), wz(p, w, a.dz, a.L * a.D, a.D);
  T4<T> nx[G::R], ndt[G::R], nz[G::R], ndy[G::R];
  T bv[G::PB], cv[G::PB];
  const auto fetch = [&](int i0) {
    load_rows<G, T, VEC>(rdt, w, i0, ndt);
    load_rows<G, T, VEC>(rdy, w, i0, ndy);
    if (a.z) load_rows<G, T, VEC>(rz, w, i0, nz);
    load_states<G, T>(rC, p, w, i0, cv);
    if (!ENDS) {
      load_rows<G, T, VEC>(rx, w, i0, nx);
      load_states<G, T>(rB, p, w, i0, bv);
    }
  };
  if (tiles) fetch(w.begin + (tiles - 1) * G::TT);

  float A2[4][NS], g[4][NS], dA[4][NS], sum[4] = {0, 0, 0, 0}, dskip[4] = {0, 0, 0, 0}, dbias[4] = {0, 0, 0, 0};
  load_exponents<NS>(p, w, A2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < NS; ++n) dA[c][n] = g[c][n] = 0.0f;
  {
    float v[4];
    per_channel(a.dt_bias, w, v);
    put4(v, &s_ch[0][4 * w.j]);
    per_channel(a.skip, w, v);
    put4(v, &s_ch[1][4 * w.j]);
  }
  wave_sync();
  // g: exp(delta_{t+1} A) g_{t+1}, what reaches frame t from behind
  if (!ENDS && w.own > 0 && p.K > kOwnJoin) {
    load_plane<NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, g);
  } else if (!ENDS) {
    if (a.dh_last) load_dn<NS>(p, a.dh_last + (int64_t)w.b * a.D * a.N, w, g);
    if (w.own > 0) pass_chunks<G, NS, VEC>(p, w, p.K - 1, -1, p.K - 1 - w.chunk, A2, g);
  }

  // what the lane adds to dB and dC: one of its 2 NS sums, or none
  const int held = sum_index<2 * NS, G::J>(w.j), place = held < 0 ? -1 : held < NS ? w.s * NS + held : G::NP + w.s * NS + held - NS;
  float* const part_bc = p.part_bc + ((int64_t)w.b * p.tiles * a.G + w.tile) * a.L * (2 * G::NP);

  // the state in front of a tile
  float h0[ENDS ? 1 : 4][NS];
  const auto plane = [&](int i0) {
    if constexpr (!ENDS) load_plane<NS, VEC>(a.saved + ((int64_t)w.b * p.ns + i0 / G::TT) * G::NP * a.D, a.D, w, h0);
  };
  if (tiles) plane(w.begin + (tiles - 1) * G::TT);

  for (int k = tiles - 1; k >= 0; --k) {
    const int i0 = w.begin + k * G::TT;
    // every tile forms its lanes' addresses again: kept over the loop they would take forty registers
    asm volatile("" : "+v"(w.s), "+v"(w.j), "+v"(w.cl), "+v"(w.c0));
    const int lane = w.s * G::J + w.j;
    {
      float bias[4], dl[G::R][4];
      get4(&s_ch[0][4 * w.j], bias);
      deltas<G, T, VEC>(p, w, i0, ndt, bias, dl);
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        float dx[4], gy[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) gy[c] = (float)ndy[r][c];
        if (a.z) {
#pragma unroll
          for (int c = 0; c < 4; ++c) gy[c] *= (float)nz[r][c] * sigmoid((float)nz[r][c]);
        }
        only_own<G, VEC>(w, i0, r, gy);
        put4(dl[r], &s_dl[r * SPLIT + w.s][4 * w.j]);
        put4(gy, &s_gy[r * SPLIT + w.s][4 * w.j]);
        if (ENDS) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] += dl[r][c];
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) dx[c] = dl[r][c] * (float)nx[r][c];
          only_own<G, VEC>(w, i0, r, dx);
          put4(dx, &s_dx[r * SPLIT + w.s][4 * w.j]);
          s_raw[0][r][lane] = nx[r];
          s_raw[1][r][lane] = ndt[r];
          s_raw[2][r][lane] = ndy[r];
          if (a.z) s_raw[3][r][lane] = nz[r];
        }
      }
      if (!ENDS) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const float v[4] = {h0[0][n], h0[1][n], h0[2][n], h0[3][n]};
          put4(v, &s_h[n][4 * lane]);
        }
      }
    }
    put_states<G, T>(p, w, i0, cv, &s_C[0][0]);
    if (!ENDS) put_states<G, T>(p, w, i0, bv, &s_B[0][0]);
    if (k) fetch(i0 - G::TT);
    wave_sync();
    int row = 4 * w.j, state = w.s * NS;
    Step<NS> f[2];
    if constexpr (ENDS) {
#pragma unroll
      for (int t = G::TT; t >= 0; --t) {
        if (t > 0) f[(t - 1) % 2].template get<G, false, true, true>(row, state, t - 1, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
        if (t == G::TT) continue;
        const Step<NS>& q = f[t % 2];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int n = 0; n < NS; ++n) g[c][n] = exp2_hw(q.dl[c] * A2[c][n]) * fmaf(q.C[n], q.gy[c], g[c][n]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // the last TB frames first: their states from the tile's start, those of the frames in front not kept
#pragma unroll 1
      for (int t0 = G::TT - TB; t0 >= 0; t0 -= TB) {
        float h[4][NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float v[4];
          get4(&s_h[n][4 * lane], v);
#pragma unroll
          for (int c = 0; c < 4; ++c) h[c][n] = v[c];
        }
#pragma unroll 1
        for (int t = 0; t < t0; ++t) {
          Step<NS> q;
          q.template get<G, true, false, false>(4 * w.j, w.s * NS, t, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int n = 0; n < NS; ++n) h[c][n] = fmaf(exp2_hw(q.dl[c] * A2[c][n]), h[c][n], q.dx[c] * q.B[n]);
        }
        float P[TB][4][NS];  // exp(delta_t A) h_{t-1}
        float dC[EARLY ? TB : 1][NS];
        row = t0 * G::CW + 4 * w.j;
        state = t0 * G::NP + w.s * NS;
        f[0].template get<G, true, EARLY, true>(row, state, 0, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
#pragma unroll
        for (int i = 0; i < TB; ++i) {
          const Step<NS>& q = f[i % 2];
          if (i + 1 < TB) f[(i + 1) % 2].template get<G, true, EARLY, true>(row, state, i + 1, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
          float y[4];
#pragma unroll
          for (int n = 0; EARLY && n < NS; ++n) dC[i][n] = 0.0f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            y[c] = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
              P[i][c][n] = exp2_hw(q.dl[c] * A2[c][n]) * h[c][n];
              h[c][n] = fmaf(q.dx[c], q.B[n], P[i][c][n]);
              y[c] = fmaf(q.C[n], h[c][n], y[c]);
              if (EARLY) dC[i][n] = fmaf(q.gy[c], h[c][n], dC[i][n]);
            }
          }
          put_sums<SPLIT>(y, w.s, s_y[0] + row + i * G::CW);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (t0 == 0 && k) plane(i0 - G::TT);  // the next tile's state takes the registers that h leaves
        // Everything is read again, and the decays are formed again: kept from above they would take more registers than there
        // are.  The compiler does not know that these are the same places.
        asm volatile("" : "+v"(row), "+v"(state));
        f[(TB - 1) % 2].template get<G, true, true, true>(row, state, TB - 1, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
#pragma unroll
        for (int i = TB - 1; i >= 0; --i) {
          const Step<NS>& q = f[i % 2];
          if (i > 0) f[(i - 1) % 2].template get<G, true, true, true>(row, state, i - 1, s_dl[0], s_dx[0], s_gy[0], s_B[0], s_C[0]);
          float S1[4], S2[4], v[2 * NS];
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            v[n] = 0.0f;
            v[NS + n] = EARLY ? dC[EARLY ? i : 0][n] : 0.0f;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            S1[c] = S2[c] = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
              const float gt = fmaf(q.C[n], q.gy[c], g[c][n]), gp = gt * P[i][c][n];
              v[n] = fmaf(gt, q.dx[c], v[n]);
              if (!EARLY) v[NS + n] = fmaf(q.gy[c], fmaf(q.dx[c], q.B[n], P[i][c][n]), v[NS + n]);
              S1[c] = fmaf(gt, q.B[n], S1[c]);
              S2[c] = fmaf(gp, A2[c][n], S2[c]);
              dA[c][n] = fmaf(gp, q.dl[c], dA[c][n]);
              g[c][n] = exp2_hw(q.dl[c] * A2[c][n]) * gt;
            }
          }
          put_sums<SPLIT>(S1, w.s, s_1[0] + row + i * G::CW);
          put_sums<SPLIT>(S2, w.s, s_gy[0] + row + i * G::CW);
          const float value = sum_lanes<2 * NS, G::J>(v, w.j);
          if (place >= 0 && i0 + t0 + i < w.own) part_bc[(int64_t)row_of(p, w.own, i0 + t0 + i) * (2 * G::NP) + (uint32_t)place] = value;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    wave_sync();
    if constexpr (!ENDS) {
      float bias[4], skip[4];
      get4(&s_ch[0][4 * w.j], bias);
      get4(&s_ch[1][4 * w.j], skip);
#pragma unroll
      for (int r = 0; r < G::R; ++r) {
        const int row = r * SPLIT + w.s;
        if (i0 + row < w.own) {
          const T4<T> x = s_raw[0][r][lane], dt = s_raw[1][r][lane], dy = s_raw[2][r][lane];
          float s1[4], s2[4], dl[4], gy[4], v[4];
          get4(&s_1[row][4 * w.j], s1);
          get4(&s_gy[row][4 * w.j], s2);
          get4(&s_dl[row][4 * w.j], dl);
#pragma unroll
          for (int c = 0; c < 4; ++c) gy[c] = (float)dy[c];
          if (a.z) {
            const T4<T> z = s_raw[3][r][lane];
            float y[4];
            get4(&s_y[row][4 * w.j], y);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float zc = (float)z[c], sg = sigmoid(zc);
              v[c] = gy[c] * fmaf(skip[c], (float)x[c], y[c]) * sg * fmaf(zc, 1.0f - sg, 1.0f);
              gy[c] *= zc * sg;
            }
            store_row<G, T, VEC>(wz, w, i0, r, v);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[c] = fmaf(dl[c], s1[c], skip[c] * gy[c]);
            dskip[c] = fmaf(gy[c], (float)x[c], dskip[c]);
          }
          store_row<G, T, VEC>(wx, w, i0, r, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = fmaf((float)x[c], s1[c], kLn2 * s2[c]);
          if (a.softplus) {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] *= sigmoid((float)dt[c] + bias[c]);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) dbias[c] += v[c];
          store_row<G, T, VEC>(wdt, w, i0, r, v);
        }
      }
      wave_sync();
    }
  }
  wave_sync();
  if (ENDS) {
    store_plane<NS, VEC>(p.chunk_h + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, g);
    put_sums<SPLIT>(sum, w.s, &s_dl[0][4 * w.j]);
    wave_sync();
    if (w.s == 0) {
      float v[4];
      get4(&s_dl[0][4 * w.j], v);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] *= 0.5f;
      store_n<float, 4, VEC>(p.chunk_s + ((int64_t)w.b * p.K + w.chunk) * a.D + w.c0, w.nc, v);
    }
    return;
  }
  if (a.dh0 && w.chunk == 0) store_dn<NS>(a.dh0 + (int64_t)w.b * a.D * a.N, a.N, w, g);
  store_plane<NS, VEC>(p.part_a + ((int64_t)w.b * p.K + w.chunk) * G::NP * a.D, a.D, w, dA);
  put_sums<SPLIT>(dskip, w.s, &s_1[0][4 * w.j]);
  put_sums<SPLIT>(dbias, w.s, &s_gy[0][4 * w.j]);
  wave_sync();
  if (w.s == 0) {
    float u[4], v[4];
    get4(&s_1[0][4 * w.j], u);
    get4(&s_gy[0][4 * w.j], v);
    float* to = p.part_d + ((int64_t)w.b * p.K + w.chunk) * 2 * a.D;
    store_n<float, 4, VEC>(to + w.c0, w.nc, u);
    store_n<float, 4, VEC>(to + a.D + w.c0, w.nc, v);
  }
}

// dB and dC: the waves' sums over their channels, added over a group's channel tiles in order, rounded once.  A value a thread, or
// several where there are more than a grid has threads.
template <class T>
__global__ void __launch_bounds__(256) scan_bc_kernel(const ScanParams p, int NP) {
  const sed_scan_args& a = p.a;
  const int64_t all = a.B * a.G * a.L * 2 * NP;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int e = (int)(i % (2 * NP)), n = e % NP;
    const int64_t r = i / (2 * NP), t = r % a.L, g = r / a.L % a.G, b = r / a.L / a.G;
    if (n >= a.N) continue;
    const bool in = !a.frames || t < a.frames[b];
    float v = 0.0f;
    if (in) {
      const float* q = p.part_bc + ((b * a.G + g) * p.tiles * a.L + t) * (2 * NP) + e;
      for (int k = 0; k < p.tiles; ++k) v += q[(int64_t)k * a.L * 2 * NP];
    }
    static_cast<T*>(e < NP ? a.dB : a.dC)[((b * a.L + t) * a.G + g) * a.N + n] = (T)v;
  }
}

// dA [D][N], d skip and d dt_bias [D]: sums over clips and chunks; dA's partial sums lie [NP][D].
__global__ void __launch_bounds__(1024) scan_param_kernel(const ScanParams p, int64_t rows_a, int64_t step_a, int64_t rows_d, int64_t step_d) {
  const sed_scan_args& a = p.a;
  const int64_t i = (int64_t)blockIdx.x * kColumns + threadIdx.x % kColumns, d = i % a.D, n = i / a.D;
  const bool live = n < a.N + 2;
  const float* q = n < a.N ? p.part_a + n * a.D + d : p.part_d + (n - a.N) * a.D + d;
  const float sum = column_sum(q, n < a.N ? rows_a : rows_d, n < a.N ? step_a : step_d, live);
  if (threadIdx.x >= kColumns || !live) return;
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
    static_cast<T*>(a.y)[b * a.D + d] = rounded<T>(y);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// Instance of a state count: NS states a lane, SPLIT lanes a channel.  The thin ones, for the forward pass, have four times the
// waves with a quarter of the states each (two of eight at 3 and 4 states).
struct Shape { int NS, SPLIT, NP, CW, TT, TS; };
Shape shape_of(int N, bool thin) {
  const auto make = [](int NS, int SPLIT) {
    const int NP = NS * SPLIT;
    return Shape{NS, SPLIT, NP, 256 / SPLIT, SPLIT == 16 ? 16 : SPLIT >= 4 ? 8 : 4, NP >= 8 ? 8 : 4};
  };
  if (N <= 1) return make(1, 1);
  if (N <= 4) return thin ? make(1, 4) : make(2, 2);
  if (N <= 8) return thin ? make(1, 8) : make(2, 4);
  if (N <= 16) return thin ? make(1, 16) : make(4, 4);
  return thin ? make(2, 16) : make(4, 8);
}

struct Layout {
  bool thin;
  int32_t K, tiles, ns;
  int64_t h, s, bc, pa, pd, total;  // float offsets into the workspace
};

// Waves of the main pass that the card holds at once.  The gradient of 16 states in fp32 is the one that LDS keeps from its two a vector
// unit (7 a compute unit): taken for 8, the last waves ran alone (1 x 16385 x 384: 230 us, 186 so; 16 x 513 x 1536: 365, 323).
int resident(const Shape& s, bool back, int size) {
  const int group = back && size == 4 ? 1 : 4, fit = 160 * 1024 / (group * lds_of(s.NS, s.SPLIT, s.NP, s.TT, back, size));
  return 256 * std::min(4 * per_unit(s.SPLIT, back), group * std::max(1, fit));
}

// Time of `waves` waves on 1024 vector units that hold `held` of them at once, in issue slots of a full unit (4.4 cycles): a wave
// takes `fixed` slots and `work`, or half of that on average where clips have lengths of their own.  Waves share a unit's slots
// (one alone gets 55 % of them, two 79 %, three 86 %, four 90 %, measured on multiply-adds), and a round is over with its last
// wave; waves of different lengths fill each other's gaps up to the last ones.
double pass_time(double waves, int held, double fixed, double work, bool ragged) {
  static const double together[] = {0.0, 1.82, 2.53, 3.49, 4.44};
  const int most = (held + 1023) / 1024;
  if (ragged) {
    const double mean = fixed + 0.5 * work;
    return std::max((fixed + work) * together[1], mean * (waves / held * together[most] + 0.5 * together[most]));
  }
  const int64_t rounds = (int64_t)waves / held, rest = (int64_t)waves % held;
  return (fixed + work) * ((double)rounds * together[most] + together[(rest + 1023) / 1024]);
}

// Chunks of a clip, and the time of the passes.  A chunk's frames are walked twice (for its end state, then for its outputs), so
// a clip stays whole where there are waves enough; else the count that pass_time gives least for.  Slots of a frame: 6 a state
// and 14 for its sums and loads, 5 and 8 without outputs, 26.5 a state in the gradient, 40 / SPLIT for forming its rows; of a
// wave's start: 500 (mostly latency); of joining a chunk: 7.5 a state and 30; of a launch: 1100 (2 us); of a chunk's states in a
// joining launch: 0.1 a state (12 bytes of traffic).
int64_t chunks_of(const sed_scan_args& a, const Shape& s, int64_t waves, int64_t nt, bool back, double& best) {
  const int n = 4 * s.NS;
  const double rows = 40.0 / s.SPLIT, main = s.TT * ((back ? 26.5 * n : 6.0 * n + 14) + rows), ends = s.TT * (5.0 * n + 8 + rows);
  const int held = resident(s, back, a.dtype == SED_F32 ? 4 : 2);
  const bool ragged = a.frames != nullptr;
  const int64_t most = std::max<int64_t>(1, nt / 2);
  int64_t K = 1;
  const auto look = [&](int64_t k) {
    const double tiles = (double)((nt + k - 1) / k), join = k > kOwnJoin ? 0.0 : (double)k * (7.5 * n + 30);
    double t = pass_time((double)(waves * k), held, 500 + join, tiles * main, ragged);
    if (k > 1) t += pass_time((double)(waves * (k - 1)), 4096, 500, tiles * ends, ragged) + 1100;
    if (k > kOwnJoin) t += 1100 + 2700 + 0.1 * n * (double)(waves * k);
    if (k == 1 || t < best) best = t, K = k;
  };
  for (int64_t k = 1; k <= most && (k == 1 || waves * k <= 16384); k += k < 32 ? 1 : k / 8) look(k);
  if (waves > 0 && held / waves > 1) look(std::min(most, held / waves));  // as many as fill the card once
  return K;
}

Layout layout_of(const sed_scan_args& a, bool back) {
  Layout l{};
  const int64_t cg = a.D / a.G;
  Shape s{};
  double best = 0.0;
  for (const bool thin : {false, true}) {
    if (thin && (back || a.N <= 1)) continue;
    const Shape c = shape_of(a.N, thin);
    const int32_t tiles = (int32_t)((cg + c.CW - 1) / c.CW), nt = (int32_t)((a.L + c.TT - 1) / c.TT);
    double t;
    const int64_t K = chunks_of(a, c, a.B * a.G * tiles, nt, back, t);
    if (best == 0.0 || t < best) best = t, s = c, l.thin = thin, l.tiles = tiles, l.K = (int32_t)K;
  }
  l.ns = (int32_t)((a.L + s.TS - 1) / s.TS);
  const int64_t K = l.K;
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
  if (!a || a->B < 0 || a->L < 0 || a->L > 0x7fffff00 || a->D < 1 || a->D > (1 << 24) || a->N < 1 || a->N > 32 || a->G < 1 || a->D % a->G) return SED_ERR_BAD_ARG;
  if (a->dtype != SED_F32 && a->dtype != SED_BF16 && a->dtype != SED_F16) return SED_ERR_BAD_ARG;
  if (a->B > 0 && a->L > 0 && (!a->x || !a->dt || !a->A || !a->Bm || !a->Cm)) return SED_ERR_BAD_ARG;
  for (const int64_t t : {a->x_t, a->dt_t, a->z_t, a->dy_t, a->Bm_t, a->Cm_t})
    if (a->L > 1 && (t < 0 || t > (1 << 26))) return SED_ERR_CAPACITY;
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

template <class G, bool BACK>
void launch_join(const ScanParams& p, hipStream_t stream) {
  if (p.K <= kOwnJoin) return;
  const int64_t n = p.a.B * G::NP * p.a.D;
  chunk_join_kernel<G, BACK><<<(unsigned)((n + 15) / 16), 1024, 0, stream>>>(p);
}

template <int NS, int SPLIT, class T, bool VEC, bool BACK>
int launch(const ScanParams& p, hipStream_t stream) {
  using G = Geo<NS, SPLIT>;
  const sed_scan_args& a = p.a;
  const int64_t waves = a.B * p.K * a.G * p.tiles, joins = p.K > kOwnJoin ? a.B * G::NP * a.D / 16 : 0;
  if (!grid_fits(waves + 4, 64) || !grid_fits(joins + 1, 1024)) return SED_ERR_CAPACITY;
  constexpr int WE = waves_of<T, BACK, true>(), WM = waves_of<T, BACK, false>();  // of the ends, of the main pass
  const unsigned ends = (unsigned)((waves + WE - 1) / WE), main = (unsigned)((waves + WM - 1) / WM);
  if constexpr (!BACK) {
    if (p.K > 1) {
      scan_forward_kernel<NS, SPLIT, T, VEC, true><<<ends, 64 * WE, 0, stream>>>(p);
      launch_join<G, false>(p, stream);
    }
    scan_forward_kernel<NS, SPLIT, T, VEC, false><<<main, 64 * WM, 0, stream>>>(p);
  } else {
    const int64_t bc = std::min<int64_t>((a.B * a.G * a.L * 2 * G::NP + 255) / 256, 1 << 23), pr = ((a.N + 2) * a.D + kColumns - 1) / kColumns;
    if (!grid_fits(pr, 1024)) return SED_ERR_CAPACITY;
    if (p.K > 1) {
      scan_backward_kernel<NS, SPLIT, T, VEC, true><<<ends, 64 * WE, 0, stream>>>(p);
      launch_join<G, true>(p, stream);
    }
    scan_backward_kernel<NS, SPLIT, T, VEC, false><<<main, 64 * WM, 0, stream>>>(p);
    scan_bc_kernel<T><<<(unsigned)bc, 256, 0, stream>>>(p, G::NP);
    int64_t rows_a = a.B * p.K, step_a = G::NP * a.D, rows_d = rows_a, step_d = 2 * a.D;
    fold_rows(p.part_a, rows_a, step_a, a.N * a.D, stream);
    fold_rows(p.part_d, rows_d, step_d, 2 * a.D, stream);
    scan_param_kernel<<<(unsigned)pr, 1024, 0, stream>>>(p, rows_a, step_a, rows_d, step_d);
  }
  return seq_status(hipGetLastError());
}

template <int NS, int SPLIT, class T, bool BACK>
int launch_v(const ScanParams& p, bool vec, hipStream_t s) {
  return vec ? launch<NS, SPLIT, T, true, BACK>(p, s) : launch<NS, SPLIT, T, false, BACK>(p, s);
}
template <int NS, int SPLIT, bool BACK>
int launch_t(const ScanParams& p, bool vec, hipStream_t s) {
  if (p.a.dtype == SED_F32) return launch_v<NS, SPLIT, float, BACK>(p, vec, s);
  if (p.a.dtype == SED_BF16) return launch_v<NS, SPLIT, bf16, BACK>(p, vec, s);
  return launch_v<NS, SPLIT, f16, BACK>(p, vec, s);
}

int run(const sed_scan_args* args, bool back, void* stream) {
  ScanParams p{};
  p.a = *args;
  if (p.a.L == 1) p.a.x_t = p.a.dt_t = p.a.z_t = p.a.dy_t = p.a.Bm_t = p.a.Cm_t = 0;  // of a single row any distance, so none that the kernels could form
  const Layout l = layout_of(p.a, back);
  if (l.total > 0 && (!args->ws || args->ws_bytes < l.total * 4 || !aligned(args->ws, 16))) return SED_ERR_CAPACITY;
  float* ws = static_cast<float*>(args->ws);
  p.K = l.K;
  p.ns = l.ns;
  p.four = p.a.N % 4 == 0 && aligned(p.a.A, 16) && aligned(p.a.h0, 16) && aligned(p.a.dh_last, 16);
  p.tiles = l.tiles;
  p.chunk_h = ws + l.h;
  p.chunk_s = ws + l.s;
  p.part_bc = ws + l.bc;
  p.part_a = ws + l.pa;
  p.part_d = ws + l.pd;
  const bool vec = vector_rows(p.a, back);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int NP = shape_of(p.a.N, l.thin).NP;
  if (back) {
    if (NP == 1) return launch_t<1, 1, true>(p, vec, s);
    if (NP == 4) return launch_t<2, 2, true>(p, vec, s);
    if (NP == 8) return launch_t<2, 4, true>(p, vec, s);
    if (NP == 16) return launch_t<4, 4, true>(p, vec, s);
    return launch_t<4, 8, true>(p, vec, s);
  }
  if (NP == 1) return launch_t<1, 1, false>(p, vec, s);
  if (NP == 4) return l.thin ? launch_t<1, 4, false>(p, vec, s) : launch_t<2, 2, false>(p, vec, s);
  if (NP == 8) return l.thin ? launch_t<1, 8, false>(p, vec, s) : launch_t<2, 4, false>(p, vec, s);
  if (NP == 16) return l.thin ? launch_t<1, 16, false>(p, vec, s) : launch_t<4, 4, false>(p, vec, s);
  return l.thin ? launch_t<2, 16, false>(p, vec, s) : launch_t<4, 8, false>(p, vec, s);
}

template <class T>
int step(const sed_scan_args& a, hipStream_t s) {
  const bool four = a.N % 4 == 0 && aligned(a.h_last, 16) && aligned(a.A, 16);
  const int need = four ? a.N / 4 : a.N, SP = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
  const int64_t grid = (a.B * a.D * SP + 255) / 256;
  if (!grid_fits(grid, 256)) return SED_ERR_CAPACITY;
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
  const sed::Shape s = sed::shape_of(N, false);
  return B * ((L + s.TS - 1) / s.TS) * s.NP * D;
}

extern "C" int64_t sed_gated_scan_workspace(const sed_scan_args* a, int32_t backward) {
  if (!a || a->B < 0 || a->L < 0 || a->D < 1 || a->N < 1 || a->N > 32 || a->G < 1 || a->D % a->G) return SED_ERR_BAD_ARG;
  // The gradient's chunks follow from the waves that LDS leaves room for, and so from the element's size where that differs: the larger
  // of both answers serves every type.
  sed_scan_args b = *a;
  b.dtype = SED_F32;
  int64_t most = sed::layout_of(b, backward != 0).total;
  const sed::Shape s = sed::shape_of(a->N, false);
  if (backward && sed::resident(s, true, 4) != sed::resident(s, true, 2)) {
    b.dtype = SED_BF16;
    most = std::max(most, sed::layout_of(b, true).total);
  }
  return most * 4;
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
