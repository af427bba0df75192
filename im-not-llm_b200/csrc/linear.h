// The linear layer's arguments and epilogue, shared by its kernels
// (linear.cu, linear_sm100.cu).
#pragma once

#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"

namespace inl {

struct LinearArgs {
  const void* x;
  const void* w;
  const float* bias;
  const void* resid;
  void* out;
  long long ldx, ldw, ldr, ldo;
  int M, N, K, act;
};

template <typename T>
__device__ __forceinline__ float load_f(const T* p) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
  else return *p;
}
template <typename T>
__device__ __forceinline__ void store_f(T* p, float v) {
  if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(v);
  else *p = v;
}

// Activations to f32 accuracy (f32 results).
__device__ __forceinline__ float act_exact(float v, int act) {
  switch (act) {
    case INL_ACT_SILU_: return v / (1.0f + expf(-v));
    case INL_ACT_GELU_ERF_: return gelu_erf_f(v);
    case INL_ACT_GELU_TANH_: return gelu_tanh_f(v);
    case INL_ACT_RELU_: return v < 0.f ? 0.f : v;  // NaN stays
    case INL_ACT_TANH_: return tanhf(v);
    default: return v;
  }
}

// gelu(x) = x Phi(x) for a result that is rounded to bf16: erfc by the rational
// form 7.1.26 of Abramowitz and Stegun (absolute error 1.5e-7), on its own side
// of zero, so that the tail of a negative x keeps its size.
__device__ __forceinline__ float gelu_erf_fast(float x) {
  const float z = fabsf(x) * 0.70710678f;
  const float t = rcp_approx(fmaf(0.3275911f, z, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * ex2_approx(z * z * -1.44269504f);  // Phi(-|x|)
  return x * (x < 0.f ? tail : 1.0f - tail);
}
// 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2 u)).
__device__ __forceinline__ float gelu_tanh_fast(float x) {
  const float u2 = x * fmaf(0.0713548162726f, x * x, 1.5957691216057f);  // 2 sqrt(2 / pi) (x + 0.044715 x^3)
  return x * rcp_approx(1.0f + ex2_approx(u2 * -1.44269504f));
}
// Activations for a result that is rounded to bf16 (half a step: 2^-9 to 2^-8
// of the value): the approximations are within 2^-20 of the argument.
__device__ __forceinline__ float act_fast(float v, int act) {
  switch (act) {
    case INL_ACT_SILU_: return silu_f(v);
    case INL_ACT_GELU_ERF_: return gelu_erf_fast(v);
    case INL_ACT_GELU_TANH_: return gelu_tanh_fast(v);
    case INL_ACT_RELU_: return v < 0.f ? 0.f : v;
    case INL_ACT_TANH_: return tanhf(v);
    default: return v;
  }
}
template <typename TO>
__device__ __forceinline__ float act_for(float v, int act) {
  return sizeof(TO) == 2 ? act_fast(v, act) : act_exact(v, act);
}

// Bias, activation, residual, one rounding, for the sum v at (m, n).
template <typename TO>
__device__ __forceinline__ void linear_finish(const LinearArgs& g, float v, long long m, int n, TO* out) {
  v = act_for<TO>(v + (g.bias ? g.bias[n] : 0.f), g.act);
  if (g.resid) v += load_f(static_cast<const TO*>(g.resid) + m * g.ldr + n);
  store_f(out + m * g.ldo + n, v);
}

template <typename TO, int R>
__device__ __forceinline__ void act_rows(float4 (&v)[R], int act) {
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = make_float4(f(v[i].x), f(v[i].y), f(v[i].z), f(v[i].w));
  };
  switch (act) {
    case INL_ACT_SILU_: each([](float x) { return act_for<TO>(x, INL_ACT_SILU_); }); break;
    case INL_ACT_GELU_ERF_: each([](float x) { return act_for<TO>(x, INL_ACT_GELU_ERF_); }); break;
    case INL_ACT_GELU_TANH_: each([](float x) { return act_for<TO>(x, INL_ACT_GELU_TANH_); }); break;
    case INL_ACT_RELU_: each([](float x) { return act_for<TO>(x, INL_ACT_RELU_); }); break;
    case INL_ACT_TANH_: each([](float x) { return act_for<TO>(x, INL_ACT_TANH_); }); break;
    default: break;
  }
}

// Activation, residual, one rounding, for columns n .. n + 3 (those below N)
// of `count` <= R rows m, m + step, ... whose sums (bias included) are v.
// `wide`: out and resid take 4 columns in one access. The residual of every
// row is read before the first store.
template <typename TO, int R>
__device__ __forceinline__ void linear_finish_rows(const LinearArgs& g, float4 (&v)[R], long long m, int step,
                                                   int count, int n, bool wide) {
  act_rows<TO, R>(v, g.act);
  TO* out = static_cast<TO*>(g.out) + m * g.ldo + n;
  const TO* res = static_cast<const TO*>(g.resid);
  const long long so = step * g.ldo, sr = step * g.ldr;
  const int left = g.N - n;
  if (res) {
    res += m * g.ldr + n;
    if (wide && left >= 4) {
      if constexpr (sizeof(TO) == 4) {
        float4 q[R];
#pragma unroll
        for (int i = 0; i < R; ++i) q[i] = i < count ? *reinterpret_cast<const float4*>(res + i * sr) : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < R; ++i) v[i].x += q[i].x, v[i].y += q[i].y, v[i].z += q[i].z, v[i].w += q[i].w;
      } else {
        uint2 q[R];
#pragma unroll
        for (int i = 0; i < R; ++i) q[i] = i < count ? *reinterpret_cast<const uint2*>(res + i * sr) : make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float2 a = unpack_bf16x2(q[i].x), b = unpack_bf16x2(q[i].y);
          v[i].x += a.x, v[i].y += a.y, v[i].z += b.x, v[i].w += b.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (i >= count) break;
        v[i].x += load_f(res + i * sr);
        if (left > 1) v[i].y += load_f(res + i * sr + 1);
        if (left > 2) v[i].z += load_f(res + i * sr + 2);
        if (left > 3) v[i].w += load_f(res + i * sr + 3);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= count) break;
    TO* o = out + i * so;
    if (wide && left >= 4) {
      if constexpr (sizeof(TO) == 4) *reinterpret_cast<float4*>(o) = v[i];
      else *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[i].x, v[i].y), pack_bf16x2(v[i].z, v[i].w));
    } else {
      store_f(o, v[i].x);
      if (left > 1) store_f(o + 1, v[i].y);
      if (left > 2) store_f(o + 2, v[i].z);
      if (left > 3) store_f(o + 3, v[i].w);
    }
  }
}

// linear_sm100.cu. Both want 16-byte rows of x and w (gemm_bf16_linear_takes).
// At most 64 rows.
cudaError_t linear_skinny(const LinearArgs& g, bool out_bf16, cudaStream_t s);
// Clusters of S CTAs (1 to 8, at most ceil(K / 64)) split K.
cudaError_t linear_cluster(const LinearArgs& g, bool out_bf16, int S, int* status, cudaStream_t s);

}  // namespace inl
