// What the sequence operators (sed_scan.hip, sed_conv.hip, sed_norm.hip) share: loads and stores of several channels at a
// time in the three element types, the activations with their slopes, and cross-lane sums.  gfx950 only, 64-lane waves.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sed_hip.h"

namespace sed {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// 2^x and 1/x as the hardware has them (1 ulp; results below the normal range are zero)
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// 1 / (1 + e^-x); e^-x overflows to infinity for x < -88, whose reciprocal is the right 0
__device__ __forceinline__ float sigmoid(float x) { return rcp_hw(1.0f + exp2_hw(-kLog2e * x)); }

// ln(1 + e^x) = max(x, 0) + log1p(e), e = e^-|x| in (0, 1].  log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, so small e keep
// their relative precision; atanh(s) / s as a polynomial in s^2 on [0, 1/9], fitted for the least relative error with its
// constant term held at 1 (iteratively weighted least squares; 5.4e-9 at most).
__device__ __forceinline__ float softplus(float x) {
  const float e = exp2_hw(-kLog2e * fabsf(x));
  const float s = e * rcp_hw(2.0f + e), q = s * s;
  float p = 0.14005996f;
  p = fmaf(p, q, 0.14000902f);
  p = fmaf(p, q, 0.20010764f);
  p = fmaf(p, q, 0.33333208f);
  p = fmaf(p, q, 1.0f);
  return fmaf(2.0f * s, p, fmaxf(x, 0.0f));  // a NaN stays one through e
}

// ---- element types: fp32 arithmetic, one rounding (to nearest, ties to even) at the store ------------------------------

typedef __bf16 bf16;
typedef _Float16 f16;

// V consecutive elements as fp32.  VEC: the address is a multiple of the vector's size, one load.  Otherwise the first n.
template <class T, int V, bool VEC>
__device__ __forceinline__ void load_n(const T* p, int n, float* out) {
  if constexpr (VEC) {
    typedef T vt __attribute__((ext_vector_type(V)));
    if (n > 0) {
      const vt v = *reinterpret_cast<const vt*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = (float)v[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = i < n ? (float)p[i] : 0.0f;
  }
}

// The rounding of an output.  For fp16 the compiler would fuse the last multiply-add with the conversion where it can (which
// rounds once instead of twice): two kernels that form the same fp32 value would then differ in a rare last bit.
template <class T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, bf16)) asm("" : "+v"(v));
  return (T)v;
}

template <class T, int V, bool VEC>
__device__ __forceinline__ void store_n(T* p, int n, const float* in) {
  if constexpr (VEC) {
    typedef T vt __attribute__((ext_vector_type(V)));
    vt v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = rounded<T>(in[i]);
    if (n > 0) *reinterpret_cast<vt*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = rounded<T>(in[i]);
  }
}

// ---- activations --------------------------------------------------------------------------------------------------------

// The normal distribution's integral up to u, and e = exp(-u^2 / 2).  With x = |u| / sqrt(2) the part beyond |u| is
// exp(-x^2) erfcx(x) / 2; erfcx(x) is t P(t), t = 1 / (1 + 0.6 x), P a polynomial fitted for the least relative error on
// 0 <= x <= 10 (iteratively weighted least squares; 5.2e-7 of the value at most as it is evaluated here), half of it taken into
// the coefficients.  So the far tail keeps its digits, and the slope's exponential is the same one.
__device__ __forceinline__ float normal_cdf(float u, float& e) {
  e = exp2_hw(-0.5f * kLog2e * u * u);
  const float t = rcp_hw(fmaf(0.6f * 0.70710678118654752440f, fabsf(u), 1.0f));
  float p = 0.5f * -0.09207959473133087f;
  p = fmaf(p, t, 0.5f * 0.41193491220474243f);
  p = fmaf(p, t, 0.5f * -0.6444382667541504f);
  p = fmaf(p, t, 0.5f * 0.2837556004524231f);
  p = fmaf(p, t, 0.5f * 0.07341824471950531f);
  p = fmaf(p, t, 0.5f * 0.2915993928909302f);
  p = fmaf(p, t, 0.5f * 0.33724936842918396f);
  p = fmaf(p, t, 0.5f * 0.3385600745677948f);
  const float tail = p * t * e;
  return u < 0.0f ? tail : 1.0f - tail;  // a NaN stays one through e
}

// act(u), act'(u)
template <int ACT>
__device__ __forceinline__ float act(float u) {
  if constexpr (ACT == SED_ACT_SILU) return u * sigmoid(u);
  if constexpr (ACT == SED_ACT_RELU) return u > 0.0f ? u : (u != u ? u : 0.0f);
  if constexpr (ACT == SED_ACT_GELU) {
    float e;
    return u * normal_cdf(u, e);
  }
  return u;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float u) {
  if constexpr (ACT == SED_ACT_SILU) {
    const float s = sigmoid(u);
    return s * fmaf(u, 1.0f - s, 1.0f);
  }
  if constexpr (ACT == SED_ACT_RELU) return u > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == SED_ACT_GELU) {
    float e;
    const float cdf = normal_cdf(u, e);
    return fmaf(u * 0.39894228040143267794f, e, cdf);
  }
  return 1.0f;
}

// ---- cross-lane sums ----------------------------------------------------------------------------------------------------

// Exchanges between lane halves (32) or between neighbouring rows of 16 lanes (16), then one add: lanes whose bit is 0 get
// a's sum over the pair of lanes that differ in that bit, the others b's.
__device__ __forceinline__ float fold32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kRor8 = 0x128, kRor4 = 0x124;  // quad_perm [1,0,3,2], [2,3,0,1]; i -> 7 - i in eights; i -> i ^ 8; i -> i - 4 in sixteens
// Sum over the 16 lanes of a row, in every lane of it.
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<kXor1>(x);
  x += dpp<kXor2>(x);
  x += dpp<kHalfMirror>(x);
  x += dpp<kRor8>(x);
  return x;
}
// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float x) {
  x = row_sum(x);
  x = fold16(x, x);
  return fold32(x, x);
}

// Sum of a column of `rows` values that lie `step` apart, for kColumns columns of a workgroup of 1024 threads: 16 threads a column
// take every 16th row, 8 of them on the way at once, and are added in order.  All threads call it; the sum is there for the first
// kColumns.
constexpr int kColumns = 64;
__device__ __forceinline__ float column_sum(const float* q, int64_t rows, int64_t step, bool live) {
  constexpr int H = 1024 / kColumns;
  __shared__ float s[H][kColumns];
  const int col = threadIdx.x % kColumns, row = threadIdx.x / kColumns;
  float v[8] = {};
  int64_t r = row;
  if (live) {
    for (; r + 7 * H < rows; r += 8 * H)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += q[(r + k * H) * step];
#pragma unroll
    for (int k = 0; k < 7; ++k) {  // every load is in bounds, so none waits for another's condition
      const float t = q[std::min(r + k * H, rows - 1) * step];
      v[k] += r + k * H < rows ? t : 0.0f;
    }
  }
  s[row][col] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  __syncthreads();
  float sum = 0.0f;
  if (row == 0)
#pragma unroll
    for (int k = 0; k < H; ++k) sum += s[k][col];
  return sum;
}

// Sums parts of `per` rows into the first row of each.
static __global__ void __launch_bounds__(1024) fold_rows_kernel(float* base, int64_t rows, int64_t step, int64_t cols, int64_t per) {
  const int64_t c = (int64_t)blockIdx.x * kColumns + threadIdx.x % kColumns, r0 = blockIdx.y * per;
  float* q = base + r0 * step + c;
  const float sum = column_sum(q, std::min(per, rows - r0), step, c < cols);
  if (threadIdx.x < kColumns && c < cols) *q = sum;  // behind column_sum's barrier nobody reads this part any more
}
// Many rows of few columns would keep a few workgroups busy for long: parts of them are summed in place first, and rows and step
// become those of the parts' sums (65536 rows of 80 columns: 360 us in one go).
inline void fold_rows(float* base, int64_t& rows, int64_t& step, int64_t cols, hipStream_t s) {
  const int64_t wide = (cols + kColumns - 1) / kColumns, most = std::min<int64_t>(rows / 256, 1024 / wide);
  if (rows <= 2048 || most < 2) return;
  const int64_t per = (rows + most - 1) / most, parts = (rows + per - 1) / per;
  fold_rows_kernel<<<dim3((unsigned)wide, (unsigned)parts), 1024, 0, s>>>(base, rows, step, cols, per);
  rows = parts;
  step *= per;
}

// A launch has fewer than 2^32 threads along an axis.
inline bool grid_fits(int64_t blocks, int threads) { return blocks <= (int64_t)(0xffffffffu / (unsigned)threads); }

inline int seq_status(hipError_t e) { return e == hipSuccess ? SED_OK : SED_ERR_HIP - (int)e; }

}  // namespace sed
