// The linear layer's arguments and epilogue, shared by its kernels
// (linear.cu, linear_sm100.cu, linear_f32_sm100.cu, gemm_sm100.cu).
#pragma once

#include <type_traits>
#include <utility>

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

// Phi(-y), y >= 0, to f32 accuracy relative to itself: exp(-y^2 / 2) times a
// polynomial in t = 1 / (1 + 0.4 y), the form of 7.1.26 of Abramowitz and Stegun
// with a minimax fit of its own (2^-26 of the value up to y = 14.5). The argument
// of the exponential is off by up to y^2 2^-24: gelu, over every f32 within 16 of
// zero, by 8.1 2^-24 of the value right of -2, 48 2^-24 at -8. 4253 x 2304 x 768 bf16
// to f32 32 us; with erfcf in its place 44.
__device__ __forceinline__ float normal_tail(float y) {
  const float t = rcp_approx(fmaf(0.4f, y, 1.0f));
  float p = fmaf(0.0322081447f, t, -0.176769182f);
  p = fmaf(p, t, 0.382164955f);
  p = fmaf(p, t, -0.373782307f);
  p = fmaf(p, t, 0.119218186f);
  p = fmaf(p, t, -0.0266585592f);
  p = fmaf(p, t, 0.0912594646f);
  p = fmaf(p, t, 0.133158177f);
  p = fmaf(p, t, 0.159625083f);
  p = fmaf(p, t, 0.159576029f);
  return p * t * ex2_approx(y * y * -0.72134752f);
}

// Activations for f32 results, each within some roundings of the value itself, on
// the tails too: the sums 1 + erf and 1 + tanh(u) of the gelus cancel left of zero
// (off by 4e-4 of the value at -4, by all of it at -5.5), Phi(-|x|) and 0.5 (1 +
// tanh(u)) = 1 / (1 + exp(-2 u)) do not. What is left is the exponential's argument,
// rounded: x^2 2^-24, and 5 |2 u| 2^-24. The quotient of the tanh form is
// __fdividef's, which gives zero where the value is below 2e-37; a plain one
// takes 39 us where this takes 19 if the exponential is past 2^126 in most places
// (bf16 1024 x 4096 x 1024 to f32, unscaled inputs).
__device__ __forceinline__ float act_exact(float v, int act) {
  switch (act) {
    case INL_ACT_SILU_: return v / (1.0f + expf(-v));
    case INL_ACT_GELU_ERF_: {
      const float tail = normal_tail(fabsf(v));
      return v * (v < 0.f ? tail : 1.0f - tail);
    }
    case INL_ACT_GELU_TANH_:  // -2 u = -2 sqrt(2 / pi) (v + 0.044715 v^3)
      return __fdividef(v, 1.0f + expf(v * fmaf(-0.0713548162726f, v * v, -1.5957691216057f)));
    case INL_ACT_RELU_: return v < 0.f ? 0.f : v;  // NaN stays
    case INL_ACT_TANH_: return tanhf(v);
    default: return v;
  }
}

// gelu(x) = x Phi(x) for a result that is rounded to bf16: normal_tail with a fit
// of 2^-20.6 of the value, on the tail too.
__device__ __forceinline__ float gelu_erf_fast(float x) {
  const float y = fabsf(x), t = rcp_approx(fmaf(0.265f, y, 1.0f));
  float p = fmaf(-0.0677870288f, t, 0.19527307f);
  p = fmaf(p, t, -0.0663628653f);
  p = fmaf(p, t, 0.142493308f);
  p = fmaf(p, t, 0.0829465985f);
  p = fmaf(p, t, 0.107836775f);
  p = fmaf(p, t, 0.105599836f);
  const float tail = p * t * ex2_approx(y * y * -0.72134752f);
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

// ------------------------------------------------------------------ clusters that share out K
// Each CTA's partial tile [128, BN] f32 in its shared memory: 16-byte piece q of
// a row at q ^ (row & 7) inside its 128-byte group, so that a warp writing 32
// rows of one piece and one reading a row's pieces both miss bank conflicts.
template <int BN>
__device__ __forceinline__ uint8_t* cluster_piece(uint8_t* part, int row, int q) {
  return part + row * (BN * 4) + (q >> 3) * 128 + (((q & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
// Counted up while a NaN is computed again, for the waits that this makes long
// (wait_alive). A static shared variable: its address takes no register.
__device__ __forceinline__ unsigned* redo_beat() {
  __shared__ unsigned beat;
  return &beat;
}
__device__ __forceinline__ unsigned redo_beats() { return *reinterpret_cast<const volatile unsigned*>(redo_beat()); }

// A plain f32 sum, ended by the first NaN. BEAT: others wait for it (redo_beat).
template <bool BEAT>
__device__ __forceinline__ float plain_dot(const LinearArgs& g, long long m, long long n) {
  const float* x = static_cast<const float*>(g.x) + m * g.ldx;
  const float* w = static_cast<const float*>(g.w) + n * g.ldw;
  float s = 0.f;
  for (int k = 0; k < g.K && !isnan(s); ++k) {
    s = fmaf(x[k], w[k], s);
    if (BEAT && (k & 0xfff) == 0) atomicAdd(redo_beat(), 1u);
  }
  return s;
}

// The NaNs among the sums v of row m, columns n .. n + 3, again.
template <bool BEAT>
__device__ __forceinline__ void redo4(const LinearArgs& g, float4& v, long long m, int n) {
  if (isnan(v.x)) v.x = plain_dot<BEAT>(g, m, n);
  if (isnan(v.y) && n + 1 < g.N) v.y = plain_dot<BEAT>(g, m, n + 1);
  if (isnan(v.z) && n + 2 < g.N) v.z = plain_dot<BEAT>(g, m, n + 2);
  if (isnan(v.w) && n + 3 < g.N) v.w = plain_dot<BEAT>(g, m, n + 3);
}

// A wait whose limit starts anew whenever redo_beat has moved: what it waits for
// may be behind a lane that computes NaNs again, for as long as K is.
__device__ __forceinline__ bool wait_alive(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  unsigned seen = redo_beats();
  uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mbar_try_wait_sleep(bar, parity, 100000u)) return true;
    if (globaltimer_ns() - t0 > INL_WAIT_TIMEOUT_NS) {
      const unsigned now = redo_beats();
      if (now == seen) {
        if (status) atomicCAS(status, 0, code);
        return false;
      }
      seen = now;
      t0 = globaltimer_ns();
    }
  }
}

// After a cluster barrier: 256 threads (tid) of each of the S CTAs sum their
// share of the tile over the cluster's partial tiles, in rank order, and run
// the epilogue on it. A thread keeps one 4-column piece; the CTAs take its rows
// in turn, four rows (4 S loads) in flight at a time. REDO: a NaN is computed
// again as a plain f32 sum.
template <typename TO, int BN, bool REDO>
__device__ __forceinline__ void cluster_finish(const LinearArgs& g, uint8_t* part, int tid, int rank, int S, int m0,
                                               int n0, bool wide) {
  constexpr int Q = BN / 4, STEP = 256 / Q;
  const int q = tid % Q, n = n0 + 4 * q, rows = min(128, g.M - m0);
  if (n >= g.N) return;
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = g.bias && n + i < g.N ? __ldg(g.bias + n + i) : 0.f;
  const uint32_t mine = smem_u32(part);
  for (int r0 = rank * STEP + tid / Q; r0 < rows; r0 += 4 * S * STEP) {
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < S; ++s) {
      const uint32_t base = mapa_shared(mine, s);
      float4 p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = min(r0 + i * S * STEP, rows - 1);
        p[i] = ld_cluster_f4(base + static_cast<uint32_t>(cluster_piece<BN>(part, row, q) - part));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i].x += p[i].x, v[i].y += p[i].y, v[i].z += p[i].z, v[i].w += p[i].w;
    }
    const int count = min(4, (rows - r0 + S * STEP - 1) / (S * STEP));
    if constexpr (REDO) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= count || !isnan(v[i].x + v[i].y + v[i].z + v[i].w)) continue;
        redo4<false>(g, v[i], m0 + r0 + i * S * STEP, n);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i].x += bias[0], v[i].y += bias[1], v[i].z += bias[2], v[i].w += bias[3];
    linear_finish_rows<TO, 4>(g, v, m0 + r0, S * STEP, count, n, wide);
  }
}

// The epilogue of 32 rows x 32 columns (corner m, n) of one warp, thread = row, v
// its sums: turned in the warp's 4 KB at `buf` (16-byte piece j of row r at j ^ (r
// & 7): no bank conflicts on either side) so that a row's columns are
// neighbouring lanes': 4 columns to a lane and 4 rows at a time where `wide`, else
// a column to a lane, so that rows of any alignment are read and written in
// whole runs. REDO (f32 operands): a NaN is computed again as a plain f32 sum.
// PLAIN (f32 results without an activation's special functions): the bias and 4
// PLAIN rows of the residual are asked for before the turn. bf16 to f32 with a
// residual: 16384 x 1024 x 512 47.6 -> 34.9 us (PLAIN 8), 65536 x 768 x 768, K in
// parts, 144 -> 124 (4: the 192- and 256-wide kernels, whose sums are 96 and 128
// registers, spill 29 and 222 words; 8: 130); beside gelu 37 -> 45.
template <typename TO, bool REDO, int PLAIN = 0>
__device__ __forceinline__ void warp_finish32(const LinearArgs& g, uint8_t* buf, const float* v, int m, int n, int lane,
                                              bool wide) {
  auto turn = [&] {
    __syncwarp();  // what was there before has been read
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    __syncwarp();
  };
  const int rows = min(32, g.M - m);
  if constexpr (PLAIN > 0) {
    if (wide && n + 32 <= g.N) {
      const int q = lane & 7, r = lane >> 3, col = n + 4 * q;
      float4 t[PLAIN], d[PLAIN], b = make_float4(0.f, 0.f, 0.f, 0.f);
      if (g.bias) {
        const float* p = g.bias + col;
        b = make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
      }
      const float* res = static_cast<const float*>(g.resid) + (m + r) * g.ldr + col;
      float* out = static_cast<float*>(g.out) + (m + r) * g.ldo + col;
      auto ahead = [&](int r0) {
#pragma unroll
        for (int i = 0; i < PLAIN; ++i, res += 4 * g.ldr)
          d[i] = r0 + r + 4 * i < rows ? *reinterpret_cast<const float4*>(res) : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      if (g.resid) ahead(0);
      turn();
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 4 * PLAIN) {
#pragma unroll
        for (int i = 0; i < PLAIN; ++i) {
          const int rr = r0 + r + 4 * i;
          t[i] = *reinterpret_cast<const float4*>(buf + rr * 128 + ((q ^ (rr & 7)) << 4));
          t[i].x += b.x, t[i].y += b.y, t[i].z += b.z, t[i].w += b.w;
        }
        if (g.act == INL_ACT_RELU_) act_rows<float, PLAIN>(t, INL_ACT_RELU_);
        if (g.resid) {
#pragma unroll
          for (int i = 0; i < PLAIN; ++i) t[i].x += d[i].x, t[i].y += d[i].y, t[i].z += d[i].z, t[i].w += d[i].w;
          if (r0 + 4 * PLAIN < 32) ahead(r0 + 4 * PLAIN);
        }
#pragma unroll
        for (int i = 0; i < PLAIN; ++i, out += 4 * g.ldo)
          if (r0 + r + 4 * i < rows) *reinterpret_cast<float4*>(out) = t[i];
      }
      return;
    }
  }
  turn();
  if (wide || REDO) {
    const int q = lane & 7, col = n + 4 * q;
    if (col >= g.N) return;
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = g.bias && col + i < g.N ? __ldg(g.bias + col + i) : 0.f;
#pragma unroll 1
    for (int r = lane >> 3; r < rows; r += 16) {
      const int count = min(4, (rows - r + 3) / 4);
      float4 t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = r + 4 * i;
        t[i] = *reinterpret_cast<const float4*>(buf + rr * 128 + ((q ^ (rr & 7)) << 4));
        if (REDO && isnan(t[i].x + t[i].y + t[i].z + t[i].w) && i < count) redo4<true>(g, t[i], m + rr, col);
        t[i].x += b[0], t[i].y += b[1], t[i].z += b[2], t[i].w += b[3];
      }
      linear_finish_rows<TO, 4>(g, t, m + r, 4, count, col, wide);
    }
  } else {
    const int col = n + lane;
    if (col >= g.N) return;
    const float b = g.bias ? __ldg(g.bias + col) : 0.f;
    const TO* res = g.resid ? static_cast<const TO*>(g.resid) + m * g.ldr + col : nullptr;
    TO* out = static_cast<TO*>(g.out) + m * g.ldo + col;
    const uint8_t* from = buf + (lane & 3) * 4;
    const int piece = lane >> 2;
    // eight rows: their residuals are read before the first is stored
    auto eight = [&](int r0, auto every) {
      constexpr bool EVERY = decltype(every)::value;
      float4 t[2];
      float* w = reinterpret_cast<float*>(t);
      float q[8];
      if (res) {
#pragma unroll
        for (int i = 0; i < 8; ++i, res += g.ldr) q[i] = EVERY || r0 + i < rows ? load_f(res) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = *reinterpret_cast<const float*>(from + (r0 + i) * 128 + ((piece ^ i) << 4)) + b;
      act_rows<TO, 2>(t, g.act);
      if (res) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] += q[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i, out += g.ldo)
        if (EVERY || r0 + i < rows) store_f(out, w[i]);
    };
    if (rows == 32) {
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += 8) eight(r0, std::true_type());
    } else {
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 8) eight(r0, std::false_type());
    }
  }
}

// Whether rows of out and resid take 4 columns in one access.
inline int linear_wide(const LinearArgs& g, bool out_bf16) {
  const uintptr_t bytes = out_bf16 ? 8 : 16;
  auto ok = [&](const void* p, long long ld) {
    return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (g.M == 1 || ld % 4 == 0);
  };
  return ok(g.out, g.ldo) && (!g.resid || ok(g.resid, g.ldr));
}

// A launch in clusters of S CTAs, allowed to start while its predecessor ends
// (launch_pdl).
template <typename... Params, typename... Args>
cudaError_t launch_cluster_pdl(void (*kern)(Params...), unsigned grid, int threads, size_t smem, int S, cudaStream_t s,
                               Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = S;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// ------------------------------------------------------------------ rows of any alignment
// Sixteen warps fetch a stage of 256 rows (128 of x, 128 of w) x 128 bytes of K,
// 16 rows each, a 4-byte word to a lane, into registers, a stage ahead. (Two
// ahead, or 32 rows to each of eight warps, spilled: the words are the registers.)
constexpr int kLoadWarps = 16, kLoadRows = 256 / kLoadWarps;

// One loading warp's rows. A bf16 row may start in the middle of a word: then
// the lanes read the words it lies in, and each takes the upper half of its own
// and the lower half of its neighbour's (the last lane's comes from `extra`,
// which lane j reads for row j). Only words with an element of the row in them
// are read; what is past K or past the matrix becomes zero. Blocks that hold
// none of that go without the checks: it is instructions that bound this.
template <typename T>
struct RowWords {
  static constexpr int E = 4 / static_cast<int>(sizeof(T));
  uintptr_t row0;  // this lane's first word in row 0
  long long step;
  int valid, K, lane;
  uint32_t shift_even, shift_odd;  // 16 where rows 0, 2, ... (1, 3, ...) start in the middle of a word

  __device__ __forceinline__ RowWords(const void* base, long long ld, int first, int rows, int K_, int lane_)
      : row0(reinterpret_cast<uintptr_t>(base) + first * ld * static_cast<long long>(sizeof(T)) + 4 * lane_),
        step(ld * static_cast<long long>(sizeof(T))),
        valid(min(rows - first, kLoadRows)),
        K(K_),
        lane(lane_),
        shift_even(static_cast<uint32_t>(row0 & 2) * 8),
        shift_odd(static_cast<uint32_t>((row0 + step) & 2) * 8) {}
  __device__ __forceinline__ bool inside(int k0) const { return valid == kLoadRows && k0 + 32 * E + 1 < K; }
  __device__ __forceinline__ uint32_t shift(int j) const { return j & 1 ? shift_odd : shift_even; }
  static __device__ __forceinline__ uint32_t word(uintptr_t at) {
    return __ldg(reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3)));
  }
  __device__ __forceinline__ void load(uint32_t (&a)[kLoadRows], uint32_t& extra, int k0) const {
    uintptr_t r = row0 + static_cast<long long>(k0) * static_cast<int>(sizeof(T));
    // row `lane`, the word after the last lane's
    const uintptr_t after = r + lane * step + 128 - 4 * lane;
    if (inside(k0)) {
      if (E == 2) extra = word(lane < kLoadRows ? after : r);
#pragma unroll
      for (int j = 0; j < kLoadRows; ++j, r += step) a[j] = word(r);
    } else {
      const int left = K - k0 - E * lane;
      if (E == 2) extra = lane < valid && shift(lane) && k0 + 63 < K ? word(after) : 0;
#pragma unroll
      for (int j = 0; j < kLoadRows; ++j, r += step)
        a[j] = j < valid && left + static_cast<int>(E == 2 ? shift(j) >> 4 : 0) > 0 ? word(r) : 0;
    }
  }
  // Whole warps: this lane's E elements of row j.
  __device__ __forceinline__ uint32_t value(const uint32_t (&a)[kLoadRows], uint32_t extra, int j) const {
    if constexpr (E == 1) return a[j];
    const uint32_t last = __shfl_sync(0xffffffffu, extra, j), next = __shfl_down_sync(0xffffffffu, a[j], 1);
    return __funnelshift_r(a[j], lane == 31 ? last : next, shift(j));
  }
  // Bits of this lane's elements of block k0 that are below K.
  __device__ __forceinline__ uint32_t mask(int k0) const {
    const int left = K - k0 - E * lane;
    return E == 1 || left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
  }
};

// The loading warps' loop over the nkb blocks of bk elements from block kb0 on:
// `put(i, j, word)` stores a word of block i, row j of the warp; `ready(i)` waits
// for block i's place in the ring and says whether to go on; `done(i)` hands it over.
template <typename T, typename Ready, typename Put, typename Done>
__device__ __forceinline__ void load_rows(const RowWords<T>& rows, int kb0, int nkb, int bk, Ready ready, Put put,
                                          Done done) {
  uint32_t a[kLoadRows], extra = 0;
  rows.load(a, extra, kb0 * bk);
  for (int i = 0; i < nkb; ++i) {
    if (!ready(i)) return;
    const int k0 = (kb0 + i) * bk;
    const uint32_t mask = rows.mask(k0);
#pragma unroll
    for (int j = 0; j < kLoadRows; ++j) put(i, j, rows.value(a, extra, j) & mask);
    if (i + 1 < nkb) rows.load(a, extra, k0 + bk);
    done(i);
  }
}

// TMEM columns [from, from + 16) of this thread's row into `total`'s (first: as
// they are), added to nearest. Whole warps.
__device__ __forceinline__ void tmem_add16(uint32_t total, uint32_t from, bool first) {
  uint32_t v[16], t[16];
  tmem_ld16(from, v);
  if (!first) tmem_ld16(total, t);
  tmem_ld_wait();
  if (!first) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(t[i]) + __uint_as_float(v[i]));
  }
  tmem_st16(total, v);
}

// linear_sm100.cu. At most 64 rows, 16-byte rows of x and w (gemm_bf16_linear_takes).
cudaError_t linear_skinny(const LinearArgs& g, bool out_bf16, cudaStream_t s);
// Clusters of S CTAs (1, 2 or 4, at most ceil(K / 64)) split K. `aligned`: 16-byte rows.
cudaError_t linear_cluster(const LinearArgs& g, bool out_bf16, bool aligned, int S, int* status, cudaStream_t s);

// linear_f32_sm100.cu: f32 operands; `takes`: 16-byte rows of x and w. S 1, 2 or
// 4, at most ceil(K / 32).
bool linear_f32_takes(const LinearArgs& g);
cudaError_t linear_f32(const LinearArgs& g, bool out_bf16, bool aligned, int S, int* status, cudaStream_t s);

}  // namespace inl
