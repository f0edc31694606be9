// Shared device helpers of the residual recurrent block's kernels (rmsnorm.hip, gated_scan.hip,
// linear.hip): storage types, vector access of a column slice, activations.
#pragma once
#include "dd_common.h"
#include "../../include/daydreamer_hip.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// largest finite e4m3 value
constexpr float E4M3_MAX = 448.0f;

// V consecutive elements as floats, and back.  The accesses are as wide as V allows whatever the address:
// global memory takes 16-byte accesses at any alignment of the element, so that rows of 1542 bf16 need
// no path of their own.
template <typename T, int V>
struct VecOf { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <int V>
__device__ __forceinline__ void load_f32(const float* p, float v[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const typename VecOf<float, 4>::type t = *reinterpret_cast<const typename VecOf<float, 4>::type*>(p + j);
      v[j] = t.x; v[j + 1] = t.y; v[j + 2] = t.z; v[j + 3] = t.w;
    }
  } else if constexpr (V == 2) {
    const typename VecOf<float, 2>::type t = *reinterpret_cast<const typename VecOf<float, 2>::type*>(p);
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
    const typename VecOf<__bf16, V>::type t = *reinterpret_cast<const typename VecOf<__bf16, V>::type*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)t[j];
  }
}
template <int V>
__device__ __forceinline__ void store_f32(float* p, const float v[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4)
      *reinterpret_cast<typename VecOf<float, 4>::type*>(p + j) = typename VecOf<float, 4>::type{v[j], v[j + 1], v[j + 2], v[j + 3]};
  } else if constexpr (V == 2) {
    *reinterpret_cast<typename VecOf<float, 2>::type*>(p) = typename VecOf<float, 2>::type{v[0], v[1]};
  } else {
    *p = v[0];
  }
}
template <int V>
__device__ __forceinline__ void store_bf16(__bf16* p, const float v[V]) {
  if constexpr (V == 1) {
    *p = (__bf16)v[0];
  } else {
    typename VecOf<__bf16, V>::type t;
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (__bf16)v[j];
    *reinterpret_cast<typename VecOf<__bf16, V>::type*>(p) = t;
  }
}
// floats of at most E4M3_MAX magnitude -> e4m3 bytes, nearest even.
template <int V>
__device__ __forceinline__ void store_e4m3(unsigned char* p, const float v[V]) {
  if constexpr (V == 8) {
    unsigned w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
      w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], t, true);
    }
    typedef unsigned u32x2 __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j], 0, false) & 0xff);
  }
}

// (the file is compiled without contraction, so that written sums stay what they are)
__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

// e^x, 1 / x to about one ulp (v_exp_f32 on x log2(e) adds |x| 2^-24 relative): every user below
// rounds to bf16 or adds terms that are larger.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// p = sigmoid(x), q = sigmoid(-x) from one exponential that cannot overflow.
__device__ __forceinline__ void sigmoid2(float x, float& p, float& q) {
  const float e = fast_exp(-fabsf(x));
  const float big = fast_rcp(1.0f + e), small = e * big;
  p = x >= 0.f ? big : small;
  q = x >= 0.f ? small : big;   // (a NaN is in both)
}

// tanh: odd polynomial where 1 - e^-2x would cancel (the first omitted term is 1e-8 relative at
// 0.3), else from the exponential.
__device__ __forceinline__ float tanh_f(float x) {
  const float a = fabsf(x), x2 = x * x;
  float s = fma_(x2, -1382.f / 155925, 62.f / 2835);
  s = fma_(x2, s, -17.f / 315); s = fma_(x2, s, 2.f / 15); s = fma_(x2, s, -1.f / 3);
  s = fma_(x * x2, s, x);
  const float e = fast_exp(-2.0f * a);
  const float l = copysignf((1.0f - e) * fast_rcp(1.0f + e), x);
  return a < 0.3f ? s : l;
}

// e^x - 1 for x <= 0: Taylor polynomial where the difference would cancel (next term 5e-9 relative).
__device__ __forceinline__ float expm1_neg(float x) {
  float s = fma_(x, 1.f / 5040, 1.f / 720);
  s = fma_(x, s, 1.f / 120); s = fma_(x, s, 1.f / 24); s = fma_(x, s, 1.f / 6); s = fma_(x, s, 0.5f); s = fma_(x, s, 1.f);
  s *= x;
  return x > -0.3f ? s : fast_exp(x) - 1.0f;
}

// Phi(-|z|), Phi(z) = (1 + erf(z / sqrt 2)) / 2, and e = exp(-z^2 / 2), with Abramowitz and Stegun's 7.1.26
// for erf (absolute error 1.5e-7, so 0.75e-7 here) on the same exponential.
__device__ __forceinline__ float normal_tail(float z, float& e) {
  const float t = fast_rcp(fma_(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
  e = __builtin_amdgcn_exp2f(-0.5f * 1.44269504088896341f * z * z);
  float q = fma_(t, 0.5f * 1.061405429f, -0.5f * 1.453152027f);
  q = fma_(t, q, 0.5f * 1.421413741f); q = fma_(t, q, -0.5f * 0.284496736f); q = fma_(t, q, 0.5f * 0.254829592f);
  return q * (e * t);
}

// out[c] (+)= sum of n partial rows: 32 columns and 32 row lanes per workgroup, eight loads in flight per
// lane, added in a fixed order (3 us for 512 x 1024; with 64 columns and 16 serial row lanes 14 us).
__global__ void __launch_bounds__(1024) k_part_sum(const float* parts, int n, int C, void* out, int type, int accumulate) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < C)
#pragma unroll 8
    for (int i = w; i < n; i += 32) t += parts[(long)i * C + c];
  sh[w][lane] = t;
  __syncthreads();
  if (w || c >= C) return;
  t = sh[0][lane];
#pragma unroll
  for (int i = 1; i < 32; ++i) t += sh[i][lane];
  if (type == DD_F32) { float* p = (float*)out + c; *p = accumulate ? *p + t : t; }
  else { __bf16* p = (__bf16*)out + c; *p = (__bf16)(accumulate ? (float)*p + t : t); }
}

// y = act(z); codes of include/daydreamer_hip.h
template <int ACT>
__device__ __forceinline__ float act_f(float z) {
  float p, q;
  if constexpr (ACT == DD_ACT_ELU) return z > 0.f ? z : expm1_neg(z);
  if constexpr (ACT == DD_ACT_SILU) { sigmoid2(z, p, q); return z * p; }
  if constexpr (ACT == DD_ACT_GELU) {   // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    p = normal_tail(z, q);
    return fma_(-fminf(fabsf(z), 3e38f), p, fmaxf(z, 0.0f));   // (infinity: 0 of it)
  }
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  float p, q;
  if constexpr (ACT == DD_ACT_ELU) return z > 0.f ? 1.0f : fast_exp(z);
  if constexpr (ACT == DD_ACT_SILU) { sigmoid2(z, p, q); return p * (1.0f + z * q); }
  if constexpr (ACT == DD_ACT_GELU) {
    p = normal_tail(z, q);
    return (z >= 0.f ? 1.0f - p : p) + z * q * 0.39894228040143268f;
  }
  return 1.0f;
}

}  // namespace
