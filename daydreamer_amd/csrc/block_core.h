// Shared device helpers of the residual recurrent block's kernels (rmsnorm.hip, gated_scan.hip,
// linear.hip): storage types, vector access of a column slice, activations.
#pragma once
#include "dd_common.h"
#include "../../include/daydreamer_hip.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// largest finite e4m3 value
constexpr float E4M3_MAX = 448.0f;

inline int dtype_size(int t) { return t == DD_F32 ? 4 : t == DD_BF16 ? 2 : 1; }

// Is every row of the [*, cols] view (p, ld) aligned to `bytes`?
inline bool rows_aligned(const void* p, long ld, int type, int bytes) {
  return p == nullptr || ((uintptr_t)p % bytes == 0 && (ld * dtype_size(type)) % bytes == 0);
}

// The first and one-past-the-last byte of a [rows, cols] view; do two of them overlap?
struct Span { uintptr_t lo, hi; };
inline Span span_of(const void* p, long rows, long ld, long cols, int type) {
  if (p == nullptr || rows <= 0 || cols <= 0) return {0, 0};
  return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)(((rows - 1) * ld + cols) * dtype_size(type))};
}
inline bool overlap(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

// V consecutive elements of type TYPE (DD_F32 / DD_BF16) as floats; p is aligned to V elements
// (at most 16 bytes).
template <int V>
__device__ __forceinline__ void load_f32(const float* p, float v[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(p + j);
      v[j] = t.x; v[j + 1] = t.y; v[j + 2] = t.z; v[j + 3] = t.w;
    }
  } else if constexpr (V == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x; v[1] = t.y;
  } else {
    v[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void load_bf16(const __bf16* p, float v[V]) {
  if constexpr (V == 1) {
    v[0] = (float)*p;
  } else {
    typedef __bf16 vec __attribute__((ext_vector_type(V)));
    const vec t = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)t[j];
  }
}
template <int V>
__device__ __forceinline__ void store_f32(float* p, const float v[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4) *reinterpret_cast<f32x4*>(p + j) = f32x4{v[j], v[j + 1], v[j + 2], v[j + 3]};
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    *p = v[0];
  }
}
template <int V>
__device__ __forceinline__ void store_bf16(__bf16* p, const float v[V]) {
  if constexpr (V == 1) {
    *p = (__bf16)v[0];
  } else {
    typedef __bf16 vec __attribute__((ext_vector_type(V)));
    vec t;
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (__bf16)v[j];
    *reinterpret_cast<vec*>(p) = t;
  }
}

// V (a multiple of 4, or 1 / 2) floats of at most E4M3_MAX magnitude -> V e4m3 bytes, nearest even.
template <int V>
__device__ __forceinline__ void store_e4m3(unsigned char* p, const float v[V]) {
  if constexpr (V % 4 == 0) {
    unsigned w[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
      w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], t, true);
    }
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
#pragma unroll
      for (int j = 0; j < V / 4; ++j) reinterpret_cast<unsigned*>(p)[j] = w[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j], 0, false) & 0xff);
  }
}

// e^x, 1 / x to about one ulp (v_exp_f32 on x log2(e) adds |x| 2^-24 relative): every user below
// rounds to bf16 or adds terms that are larger.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// p = sigmoid(x), q = sigmoid(-x) from one exponential that cannot overflow.
__device__ __forceinline__ void sigmoid2(float x, float& p, float& q) {
  const float e = fast_exp(-fabsf(x));
  const float big = fast_rcp(1.0f + e), small = e * big;
  p = x >= 0.f ? big : small;
  q = x >= 0.f ? small : big;
  if (x != x) p = q = x;
}

// tanh: odd polynomial where 1 - e^-2x would cancel (the first omitted term is 1e-8 relative at
// 0.3), else from the exponential.
__device__ __forceinline__ float tanh_f(float x) {
  const float a = fabsf(x), x2 = x * x;
  const float s = x + x * x2 * (-1.f / 3 + x2 * (2.f / 15 + x2 * (-17.f / 315 + x2 * (62.f / 2835 - x2 * (1382.f / 155925)))));
  const float e = fast_exp(-2.0f * a);
  const float l = copysignf((1.0f - e) * fast_rcp(1.0f + e), x);
  return a < 0.3f ? s : l;
}

// e^x - 1 for x <= 0: Taylor polynomial where the difference would cancel (next term 5e-9 relative).
__device__ __forceinline__ float expm1_neg(float x) {
  const float s = x * (1.f + x * (1.f / 2 + x * (1.f / 6 + x * (1.f / 24 + x * (1.f / 120 + x * (1.f / 720 + x * (1.f / 5040)))))));
  return x > -0.3f ? s : fast_exp(x) - 1.0f;
}

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2), with Abramowitz and Stegun's 7.1.26 for erf
// (absolute error 1.5e-7, so 0.75e-7 here) on the same exponential.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = fast_rcp(1.0f + 0.3275911f * 0.70710678118654752f * fabsf(z));
  e = fast_exp(-0.5f * z * z);
  const float q = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z >= 0.f ? 1.0f - q : q;
}

// y = act(z); codes of include/daydreamer_hip.h
template <int ACT>
__device__ __forceinline__ float act_f(float z) {
  float p, q;
  if constexpr (ACT == DD_ACT_ELU) return z > 0.f ? z : expm1_neg(z);
  if constexpr (ACT == DD_ACT_SILU) { sigmoid2(z, p, q); return z * p; }
  if constexpr (ACT == DD_ACT_GELU) return z * normal_cdf(z, q);
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  float p, q;
  if constexpr (ACT == DD_ACT_ELU) return z > 0.f ? 1.0f : fast_exp(z);
  if constexpr (ACT == DD_ACT_SILU) { sigmoid2(z, p, q); return p * (1.0f + z * q); }
  if constexpr (ACT == DD_ACT_GELU) { p = normal_cdf(z, q); return p + z * q * 0.39894228040143268f; }
  return 1.0f;
}

}  // namespace
