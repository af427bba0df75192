// Linear layer out = act(x w^T + bias) + resid (inl_cuda_linear): the entry
// point, the choice of the kernel, and linear_rows_kernel, the FFMA form for few
// rows of f32 operands, or of operands no vector load aligns with.
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

// V consecutive values of a row from k on, zero past K. V = 4 wants them on a 16-byte boundary.
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* row, int k, int K, float (&v)[V]) {
  if constexpr (V == 4) {
    if (K - k >= 4) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(row + k));
      v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = i < K - k ? load_f(row + k + i) : 0.f;
}

// A read of w, like linear_skinny_kernel, on FFMA: a CTA owns R rows of w and MT
// rows of x, its 8 warps take turns of K, a lane V values of each row. f32 sums:
// over a lane's share of K, then the lanes and the warps in order. One f32 row
// x 1024 x 1024: 2.6 us; x 4096 x 1024: 6.0 us = 2.8 TB/s (w in L2; 7.4 from
// memory); 4 rows of the latter 10 us, with 39 words a thread spilled at three
// CTAs an SM; 8 rows 13.5 us, bound by the loads of x, which every CTA makes again.
template <typename TX, typename TO, int MT, int R, int V>
__global__ void __launch_bounds__(256, MT < 8 ? 3 : 2) linear_rows_kernel(LinearArgs g) {
  __shared__ float red[8][MT * R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * R;
  const TX* w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) w[r] = static_cast<const TX*>(g.w) + min(n0 + r, g.N - 1) * g.ldw;
  for (int m0 = blockIdx.y * MT; m0 < g.M; m0 += gridDim.y * MT) {
    const TX* x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = static_cast<const TX*>(g.x) + min(m0 + m, g.M - 1) * g.ldx;
    float acc[MT][R] = {};
#pragma unroll(MT < 8 ? 2 : 1)
    for (int k = (warp * 32 + lane) * V; k < g.K; k += 256 * V) {
      float wv[R][V], xv[MT][V];
#pragma unroll
      for (int r = 0; r < R; ++r) load_values<TX, V>(w[r], k, g.K, wv[r]);
#pragma unroll
      for (int m = 0; m < MT; ++m) load_values<TX, V>(x[m], k, g.K, xv[m]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[m][r] = fmaf(xv[m][i], wv[r][i], acc[m][r]);
    }
    __syncthreads();  // the rows before have been summed
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float t = warp_sum(acc[m][r]);
        if (lane == 0) red[warp][m * R + r] = t;
      }
    __syncthreads();
    if (threadIdx.x < MT * R) {
      const int m = m0 + threadIdx.x / R, n = n0 + threadIdx.x % R;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += red[i][threadIdx.x];
      if (m < g.M && n < g.N) linear_finish(g, v, static_cast<long long>(m), n, static_cast<TO*>(g.out));
    }
  }
}

template <typename TX, typename TO, int MT, int V>
cudaError_t launch_rows(const LinearArgs& g, cudaStream_t s) {
  constexpr int R = 4;
  const dim3 grid((g.N + R - 1) / R, std::min((g.M + MT - 1) / MT, 65535));
  return launch_plain(linear_rows_kernel<TX, TO, MT, R, V>, grid, dim3(256), 0, s, g);
}

template <typename TX, typename TO, int V>
cudaError_t launch_rows_for(const LinearArgs& g, cudaStream_t s) {
  if (g.M == 1) return launch_rows<TX, TO, 1, V>(g, s);
  if (g.M <= 4) return launch_rows<TX, TO, 4, V>(g, s);
  return launch_rows<TX, TO, 8, V>(g, s);
}

cudaError_t linear_rows(const LinearArgs& g, bool x_bf16, bool out_bf16, bool aligned, cudaStream_t s) {
  if (x_bf16)
    return out_bf16 ? launch_rows_for<__nv_bfloat16, __nv_bfloat16, 1>(g, s)
                    : launch_rows_for<__nv_bfloat16, float, 1>(g, s);
  if (aligned)
    return out_bf16 ? launch_rows_for<float, __nv_bfloat16, 4>(g, s) : launch_rows_for<float, float, 4>(g, s);
  return out_bf16 ? launch_rows_for<float, __nv_bfloat16, 1>(g, s) : launch_rows_for<float, float, 1>(g, s);
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

// The same for the kernels with 128 x 128 tiles (f32, and rows of any
// alignment): the S of the least (waves over the SMs) x (blocks of 128 bytes of k
// + 10 for a tile's start and end), the 10 once where a CTA walks over tiles
// (f32, 16-byte rows, S = 1). Measured (us), f32, S = 1 / 2 / 4 / 8: 1024 x 1024 x
// 1024 31 / 19 / 28 / 72; 1024 x 4096 x 1024 56 / 77 / 110 / 254; 8192 x 1024 x
// 4096 385 / 386 / 501 / 816; 4253 x 768 x 768 44 / 49 / 84 / 194;
// 128 x 1024 x 1024 30 / 18 / 13 / 15.
int tile_cluster_size(const LinearArgs& g, int bk, bool walk, int sms) {
  const long long tiles = static_cast<long long>((g.M + 127) / 128) * ((g.N + 127) / 128);
  const int k_blocks = (g.K + bk - 1) / bk;
  int best = 1;
  long long least = -1;
  for (int S = 1; S <= 4 && S <= k_blocks; S *= 2) {
    const long long waves = (tiles * S + sms - 1) / sms, blocks = (k_blocks + S - 1) / S;
    const long long cost = walk && S == 1 ? waves * blocks + 10 : waves * (blocks + 10);
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
  if (g.K > 0 && (g.out == g.x || g.out == g.w)) return bad("out is neither x nor w");
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
    if (S > 1) return launched("linear", linear_cluster(g, ob, true, S, status, s));
    const int rc = gemm_bf16_linear(t, ob, s);
    if (rc == 0) return INL_OK;
    return record_error(INL_ERR_INFERENCE,
                        rc == -3 ? std::string("linear launch failed: ") + cudaGetErrorString(cudaGetLastError())
                                 : std::string("linear: no TMA map for x, w or out"));
  }
  const bool aligned = xb ? gemm_bf16_linear_takes(t) : linear_f32_takes(g);
  // Few rows, where the product is a read of w. Measured (us), linear_rows /
  // the tensor-core kernel, f32, K = 1024: M = 1, N = 4096 6.0 / 13.5; 8 x 4096
  // 13.5 / 14.1; 16 x 1024 8.1 / 10.8; 16 x 4096 23 / 14; 32 x 1024 14 / 11.4;
  // bf16 rows of odd strides: 8 x 1024 5.0 / 10.8; 32 x 1024 15 / 12.
  if (g.K == 0 || g.M <= 8 || (g.M <= 16 && g.N <= 8 * sms))
    return launched("linear", linear_rows(g, xb, ob, aligned, s));
  if (xb) return launched("linear", linear_cluster(g, ob, false, tile_cluster_size(g, 64, false, sms), status, s));
  return launched("linear", linear_f32(g, ob, aligned, tile_cluster_size(g, 32, aligned, sms), status, s));
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
