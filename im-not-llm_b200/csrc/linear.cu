// Linear layer out = act(x w^T + bias) + resid (inl_cuda_linear).
//
// linear_any_kernel takes every shape, stride and alignment: 64 x 64 outputs per
// CTA, 16-deep K slices staged in shared memory as f32, 4 x 4 outputs per
// thread on FFMA.
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "hook_checks.h"
#include "kernels.h"
#include "linear.h"

namespace inl {

namespace {

template <typename TX, typename TO>
__global__ void __launch_bounds__(256) linear_any_kernel(LinearArgs g) {
  constexpr int BM = 64, BN = 64, BK = 16;
  __shared__ float xs[BK][BM + 4];
  __shared__ float ws[BK][BN + 4];
  const TX* x = static_cast<const TX*>(g.x);
  const TX* w = static_cast<const TX*>(g.w);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n_tiles = (g.N + BN - 1) / BN;
  const long long tiles = static_cast<long long>((g.M + BM - 1) / BM) * n_tiles;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int m0 = static_cast<int>(tile / n_tiles) * BM, n0 = static_cast<int>(tile % n_tiles) * BN;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < g.K; k0 += BK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int idx = threadIdx.x + i * 256, r = idx >> 4, kk = idx & 15;
        const bool k_ok = kk < g.K - k0;
        xs[kk][r] = (k_ok && r < g.M - m0) ? load_f(x + (m0 + r) * g.ldx + k0 + kk) : 0.f;
        ws[kk][r] = (k_ok && r < g.N - n0) ? load_f(w + (n0 + r) * g.ldw + k0 + kk) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < BK; ++kk) {
        const float4 a = *reinterpret_cast<const float4*>(&xs[kk][ty * 4]);
        const float4 b = *reinterpret_cast<const float4*>(&ws[kk][tx * 4]);
        const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (ty * 4 + i >= g.M - m0) continue;
      const long long m = m0 + ty * 4 + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (tx * 4 + j >= g.N - n0) continue;
        const int n = n0 + tx * 4 + j;
        float v = act_exact(acc[i][j] + (g.bias ? g.bias[n] : 0.f), g.act);
        if (g.resid) v += load_f(static_cast<const TO*>(g.resid) + m * g.ldr + n);
        store_f(static_cast<TO*>(g.out) + m * g.ldo + n, v);
      }
    }
  }
}

template <typename TX, typename TO>
cudaError_t launch_linear_any(const LinearArgs& g, cudaStream_t s) {
  const long long tiles = static_cast<long long>((g.M + 63) / 64) * ((g.N + 63) / 64);
  linear_any_kernel<TX, TO><<<static_cast<unsigned>(std::min<long long>(tiles, 1 << 20)), 256, 0, s>>>(g);
  return cudaGetLastError();
}

int bad(const char* why) { return record_error(INL_ERR_INVALID_INPUT, std::string("linear: ") + why); }

// CTAs per cluster for a product whose 128 x 64 tiles leave SMs idle: 4 or 2
// while all of them run at once and each keeps 4 (or 3) blocks of 64 k. An SM
// takes operands from L2 at about 100 KB/us, so a lone CTA needs 0.24 us per
// block of k. Measured (us), S = 1 (the persistent kernel) / 2 / 4:
// 128 x 1024 x 1024 7.6 / 6.4 / 6.1; 256 x 768 x 768 6.5 / 5.9 / 6.2;
// 256 x 1024 x 2048 11.9 / 8.7 / 8.0; 512 x 1024 x 2048 12.2 / 9.2 / 15.6;
// 64 x 4096 x 1024 7.7 / 6.5 / 12.7. S = 8 took 11 us and more.
int cluster_size(const LinearArgs& g, int sms) {
  const long long tiles = static_cast<long long>((g.M + 127) / 128) * ((g.N + 63) / 64);
  const int k_blocks = (g.K + 63) / 64;
  if (tiles * 4 <= sms && k_blocks >= 16) return 4;
  return tiles * 2 <= sms && k_blocks >= 6 ? 2 : 1;
}

// The same for the f32 kernel, whose CTAs take one tile each: the S of the
// least (waves over the SMs) x (blocks of 32 k + 4 for a tile's start and end).
// Measured (us), S = 1 / 2 / 4 / 8: 1024 x 1024 x 1024 36 / 21 / 29 / 74;
// 1024 x 4096 x 1024 72 / 85 / 117 / 262; 8192 x 1024 x 4096 478 / 444 / 575 /
// 906; 4253 x 768 x 768 66 / 58 / 94 / 201; 32 x 1024 x 1024 40 / 22 / 15 / 12.
int f32_cluster_size(const LinearArgs& g, int sms) {
  const long long tiles = static_cast<long long>((g.M + 127) / 128) * ((g.N + 127) / 128);
  const int k_blocks = (g.K + 31) / 32;
  int best = 1;
  long long least = -1;
  for (int S = 1; S <= 8 && S <= k_blocks; S *= 2) {
    const long long cost = (tiles * S + sms - 1) / sms * ((k_blocks + S - 1) / S + 4);
    if (least < 0 || cost < least) least = cost, best = S;
  }
  return best;
}

int linear(const LinearArgs& g, int dtype, int out_dtype, int* status, cudaStream_t s) {
  if ((dtype != INL_DTYPE_F32 && dtype != INL_DTYPE_BF16) || (out_dtype != INL_DTYPE_F32 && out_dtype != INL_DTYPE_BF16))
    return bad("dtypes are f32 or bf16");
  constexpr int kMost = 1 << 30;  // tile indices and K offsets stay in 32 bits
  if (g.M < 0 || g.N < 0 || g.K < 0 || g.M > kMost || g.N > kMost || g.K > kMost)
    return bad("M, N, K from 0 to 2^30");
  if (static_cast<long long>(g.M) * g.N > (1ll << 40)) return bad("M * N at most 2^40");
  if (g.act < INL_ACT_SILU_ || g.act > INL_ACT_TANH_) return bad("unknown activation");
  if (g.M == 0 || g.N == 0) return INL_OK;
  for (long long ld : {g.ldx, g.ldw, g.ldr, g.ldo})
    if (ld > (1ll << 40)) return bad("strides below 2^40");
  if ((g.M > 1 && (g.ldx < g.K || g.ldo < g.N || (g.resid && g.ldr < g.N))) || (g.N > 1 && g.ldw < g.K))
    return bad("row strides are at least the row's width");
  if (!g.out || (g.K > 0 && (!g.x || !g.w))) return record_error(INL_ERR_CONFIG, "linear: NULL x, w or out");
  if (g.resid == g.out && g.M > 1 && g.ldr != g.ldo) return bad("out may be resid only at the same stride");
  const int es = dtype == INL_DTYPE_BF16 ? 2 : 4, eo = out_dtype == INL_DTYPE_BF16 ? 2 : 4;
  const std::initializer_list<HookPtr> ptrs = {{g.K ? g.x : nullptr, es, "x"}, {g.K ? g.w : nullptr, es, "w"},
                                               {g.bias, 4, "bias"},            {g.resid, eo, "resid"},
                                               {g.out, eo, "out"},             {status, 4, "status"}};
  int r;
  if ((r = check_aligned("linear", ptrs)) || (r = check_reachable("linear", ptrs))) return r;
  const bool xb = dtype == INL_DTYPE_BF16, ob = out_dtype == INL_DTYPE_BF16;
  GemmArgs t;
  t.A = static_cast<const __nv_bfloat16*>(g.x), t.lda = g.ldx;
  t.W = static_cast<const __nv_bfloat16*>(g.w), t.ldw = g.ldw;
  t.M = g.M, t.N = g.N, t.K = g.K, t.act = g.act, t.bias = g.bias;
  t.out = g.out, t.ldo = g.ldo, t.resid = static_cast<const __nv_bfloat16*>(g.resid), t.ldr = g.ldr;
  t.status = status;
  const int sms = num_sms_cached();
  if (xb && gemm_bf16_linear_takes(t)) {
    if (g.M <= 32 || (g.M <= 64 && g.N <= 8 * sms)) return launched("linear", linear_skinny(g, ob, s));
    const int S = cluster_size(g, sms);
    if (S > 1) return launched("linear", linear_cluster(g, ob, S, status, s));
    const int rc = gemm_bf16_linear(t, ob, s);
    if (rc == 0) return INL_OK;
    return record_error(INL_ERR_INFERENCE, rc == -3 ? "linear launch failed" : "linear: no TMA map for x, w or out");
  }
  if (!xb && linear_f32_takes(g)) return launched("linear", linear_f32(g, ob, f32_cluster_size(g, sms), status, s));
  return launched("linear", xb ? (ob ? launch_linear_any<__nv_bfloat16, __nv_bfloat16>(g, s)
                                     : launch_linear_any<__nv_bfloat16, float>(g, s))
                               : (ob ? launch_linear_any<float, __nv_bfloat16>(g, s)
                                     : launch_linear_any<float, float>(g, s)));
}

}  // namespace

}  // namespace inl

extern "C" {

int inl_cuda_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int M, int N, int K,
                    const float* bias, int act, const void* resid, int64_t ldr, void* out, int64_t ldo, int out_dtype,
                    int* status, void* stream) {
  return inl::guarded([&] {
    const inl::LinearArgs g{x, w, bias, resid, out, ldx, ldw, ldr, ldo, M, N, K, act};
    return inl::linear(g, dtype, out_dtype, status, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
