// Linear layers of few rows, out = act(x w^T + bias) + resid with bf16 operands:
// the sizes at which the persistent GEMM leaves most of the SMs idle.
//
// linear_skinny_kernel: up to 64 rows. The product is a read of w, so w goes
// from global memory straight into mma.sync fragments, with no shared memory
// in between: the k order inside a product is free as long as x and w agree, so
// a lane takes 16 contiguous bytes of its row as the k pairs (0,1 | 8,9) of one
// m16n8k16 and of the next. A CTA owns 8 NT rows of w, its 8 or 16 warps split K
// and are summed in shared memory in warp order. The tensor core truncates its
// sums, so each holds 64 to 256 of K and they are added to nearest (in one
// accumulator all along, sums of one sign were off by 8e-7 at K = 16384, by
// 3e-4 at 2^20). A read of w bounds it: one row x
// 4096 x 1024 3.2 us = 2.6 TB/s, of which launch and one trip to memory are 2.
//
// linear_cluster_kernel: some hundreds of rows, or few columns. A cluster of S
// CTAs shares one 128 x 64 tile, each with its own slice of K on tcgen05
// (TMA ring, accumulator in TMEM); the partial tiles meet in shared memory and
// every CTA sums its share of the elements over the cluster's copies, in rank
// order, and runs the epilogue on it. No workspace, no atomics, the same bits
// every time. 256 x 1024 x 2048: 8.0 us where the persistent kernel's 32 tiles
// take 11.9.
#include <algorithm>
#include <type_traits>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "kernels.h"
#include "linear.h"

namespace inl {

namespace {

// ------------------------------------------------------------------ skinny
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 bf16 of a row from element k on, zero past K (the row's last piece is
// read element by element: nothing past K is touched).
__device__ __forceinline__ uint4 load8_to(const __nv_bfloat16* row, int k, int K) {
  if (K - k >= 8) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = k + i < K ? reinterpret_cast<const uint16_t*>(row)[k + i] : 0u;
  return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}

template <typename TO, int MT, int NT, int U, int W>
__global__ void __launch_bounds__(32 * W) linear_skinny_kernel(LinearArgs g) {
  extern __shared__ float red_raw[];
  auto red = reinterpret_cast<float(*)[MT * 16][NT * 8 + 1]>(red_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * NT * 8;
  const int r = lane >> 2, kq = (lane & 3) * 8;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(g.x);
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(g.w);
  float sum[MT][NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int k0 = warp * 32; k0 < g.K; k0 += W * 32 * U) {
    float acc[MT][NT][4] = {};
    uint4 wv[U][NT], xv[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * W * 32 + kq;
      const bool k_ok = k < g.K;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = n0 + j * 8 + r;
        wv[u][j] = k_ok && n < g.N ? load8_to(w + n * g.ldw, k, g.K) : zero;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = i * 16 + r;
        xv[u][i][0] = k_ok && m < g.M ? load8_to(x + m * g.ldx, k, g.K) : zero;
        xv[u][i][1] = k_ok && m + 8 < g.M ? load8_to(x + (m + 8) * g.ldx, k, g.K) : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 lo = xv[u][i][0], hi = xv[u][i][1];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_bf16_16816(acc[i][j], lo.x, hi.x, lo.y, hi.y, wv[u][j].x, wv[u][j].y);
          mma_bf16_16816(acc[i][j], lo.z, hi.z, lo.w, hi.w, wv[u][j].z, wv[u][j].w);
        }
      }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][j][e] += acc[i][j][e];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][i * 16 + r + (e >> 1) * 8][j * 8 + (lane & 3) * 2 + (e & 1)] = sum[i][j][e];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 16 * NT * 8; o += 32 * W) {
    const int m = o / (NT * 8), c = o % (NT * 8), n = n0 + c;
    if (m >= g.M || n >= g.N) continue;
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < W; ++s) v += red[s][m][c];
    linear_finish(g, v, static_cast<long long>(m), n, static_cast<TO*>(g.out));
  }
}

template <typename TO, int MT, int NT, int U, int W>
cudaError_t launch_skinny(const LinearArgs& g, cudaStream_t s) {
  return launch_plain(linear_skinny_kernel<TO, MT, NT, U, W>, dim3((g.N + 8 * NT - 1) / (8 * NT)), dim3(32 * W),
                      W * MT * 16 * (NT * 8 + 1) * 4, s, g);
}

template <typename TO>
cudaError_t launch_skinny_for(const LinearArgs& g, cudaStream_t s) {
  // Few columns: 8 rows of w per CTA, on as many SMs as that gives. More: more
  // rows of w per CTA, so that each load of x serves them all, while about two
  // CTAs of 8 warps stay on each SM; 16 warps where an SM has one CTA.
  // Measured (us), 8 / 16 / 32 rows of w per CTA: M = 1, K = 1024: N = 1024
  // 2.8 / 2.8 / 3.5, N = 4096 5.1 / 3.2 / 3.5; M = 16, K = 768, N = 2304
  // 3.3 / 3.0 / 3.6; M = 32, K = 1024, N = 4096 6.5 / 6.8 / 5.9. 16 against 8
  // warps: M = 1, N = K = 1024 2.6 / 2.8; M = 19, N = 1024, K = 2048 4.1 / 4.7;
  // M = 1, N = 2048, K = 2048 (256 CTAs) 4.9 / 3.6.
  const int sms = num_sms_cached();
  const bool one = g.N <= 8 * sms;
  if (g.M <= 16) {
    if (one) return launch_skinny<TO, 1, 1, 4, 16>(g, s);
    if (g.N <= 14 * sms) return launch_skinny<TO, 1, 1, 8, 8>(g, s);
    if (g.N <= 28 * sms) return launch_skinny<TO, 1, 2, 4, 8>(g, s);
    return launch_skinny<TO, 1, 4, 4, 8>(g, s);
  }
  if (g.M <= 32) {
    if (one) return launch_skinny<TO, 2, 1, 4, 16>(g, s);
    if (g.N <= 14 * sms) return launch_skinny<TO, 2, 1, 4, 8>(g, s);
    return launch_skinny<TO, 2, 4, 2, 8>(g, s);
  }
  return launch_skinny<TO, 4, 1, 2, 16>(g, s);
}

// ------------------------------------------------------------------ cluster split-K
constexpr int kBM = 128, kBK = 64;
// warp 0 TMA, warp 1 MMA, warps 2..9 move the accumulator out; for rows that no
// TMA map takes, warps 10..25 load them
constexpr int threads_of(bool tma) { return 320 + (tma ? 0 : 32 * kLoadWarps); }

template <int kBN>
struct ClusterCfg {
  static constexpr int STAGES = kBN == 128 ? 4 : 6;
  static constexpr int CHUNK = 8;  // K blocks (512 of K) between promotions of the sum
  static constexpr int A_BYTES = kBM * kBK * 2, B_BYTES = kBN * kBK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PART_BYTES = kBM * kBN * 4;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + PART_BYTES + 1024 + 256;
};

// TMA: 16-byte rows, tiles of 64 columns. Else rows of any alignment, loaded word
// by word (RowWords) into the same swizzled layout, and tiles of 128 columns,
// since those loads are what bounds it: 1024 x 4096 x 1024 at odd strides 48 us
// (13 us aligned), 8192 x 1024 x 4096 272 us = 252 TFLOP/s. The same loads by
// 4-byte cp.async took 268 and 1813 us.
template <typename TO, bool TMA>
__global__ void __launch_bounds__(threads_of(TMA), 1)
    linear_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          LinearArgs g, int S, int wide, int* status) {
  constexpr int BN = TMA ? 64 : 128;
  using C = ClusterCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  uint8_t* part = sB + C::STAGES * C::B_BYTES;  // this CTA's partial tile, f32
  uint64_t* full = reinterpret_cast<uint64_t*>(part + C::PART_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / S;
  const int n_tiles = (g.N + BN - 1) / BN;
  const int m0 = tile / n_tiles * kBM, n0 = tile % n_tiles * BN;
  const int k_blocks = (g.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<long long>(k_blocks) * rank / S);
  const int nkb = static_cast<int>(static_cast<long long>(k_blocks) * (rank + 1) / S) - kb0;  // > 0: S <= k_blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], TMA ? 1 : kLoadWarps);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 8);
    }
    fence_barrier_init();
    if (TMA) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, TMA ? 2 * BN : 4 * BN);  // two accumulators (and a total: a power of two)
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();

  if (warp == 0) {
    if (TMA && lane == 0) {
      int issued = 0;
      for (; issued < nkb; ++issued) {
        const int st = issued % C::STAGES, kb = kb0 + issued;
        if (!mbar_wait(&empty[st], ((issued / C::STAGES) & 1) ^ 1, status, INL_DEV_TIMEOUT_PRODUCER)) break;
        mbar_expect_tx(&full[st], C::STAGE_BYTES);
        tma_load_2d(sA + st * C::A_BYTES, &tmA, &full[st], kb * kBK, m0);
        tma_load_2d(sB + st * C::B_BYTES, &tmB, &full[st], kb * kBK, n0);
      }
      // every copy has landed before the CTA can leave
      for (int f = max(0, issued - C::STAGES); f < issued; ++f)
        if (!mbar_wait(&full[f % C::STAGES], (f / C::STAGES) & 1, status, INL_DEV_TIMEOUT_DRAIN)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_bf16(kBM, BN);
      for (int i = 0; i < nkb; ++i) {
        const int st = i % C::STAGES, chunk = i / C::CHUNK, acc = chunk & 1;
        if (i % C::CHUNK == 0 && !mbar_wait(&tempty[acc], ((chunk >> 1) & 1) ^ 1, status, INL_DEV_TIMEOUT_MMA)) break;
        if (!mbar_wait(&full[st], (i / C::STAGES) & 1, status, INL_DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint64_t a = sw128_kmajor_desc(smem_u32(sA + st * C::A_BYTES));
        const uint64_t b = sw128_kmajor_desc(smem_u32(sB + st * C::B_BYTES));
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk)
          umma_bf16(tmem + acc * BN, a + static_cast<uint64_t>(kk * 2), b + static_cast<uint64_t>(kk * 2), idesc,
                    (i % C::CHUNK != 0 || kk != 0) ? 1u : 0u);
        umma_commit(&empty[st]);
        if (i % C::CHUNK == C::CHUNK - 1 || i == nkb - 1) umma_commit(&tfull[acc]);
      }
    }
  } else if (warp < 10) {
    // thread = tile row (lane quadrant warp % 4), half of the columns. The
    // tensor core's accumulator truncates (1e-6 of the sum, toward zero, by K =
    // 1024): every CHUNK blocks it is moved out and summed here, rounded to
    // nearest.
    constexpr int HW = BN / 2;
    const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * HW;
    // Sums in registers; in TMEM beside the loading warps, whose loads need them.
    constexpr int R = TMA ? HW : 16;
    float sum[R];
#pragma unroll
    for (int j = 0; j < R; ++j) sum[j] = 0.f;
    const int chunks = (nkb + C::CHUNK - 1) / C::CHUNK;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const int acc = c & 1;
      if (!(ok = mbar_wait_warp(&tfull[acc], (c >> 1) & 1, status, INL_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < HW; j += 16) {
        if constexpr (TMA) {
          uint32_t v[16];
          tmem_ld16(t_row + acc * BN + j, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[j + i] += __uint_as_float(v[i]);
        } else {
          tmem_add16(t_row + 2 * BN + j, t_row + acc * BN + j, c == 0);
        }
      }
      if constexpr (!TMA) tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
    if (ok) {
#pragma unroll
      for (int j = 0; j < HW; j += 16) {
        uint32_t t[16];
        if constexpr (!TMA) {
          tmem_ld16(t_row + 2 * BN + j, t);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float4 v;
          if constexpr (TMA)
            v = make_float4(sum[(j + 4 * i) % R], sum[(j + 4 * i + 1) % R], sum[(j + 4 * i + 2) % R], sum[(j + 4 * i + 3) % R]);
          else
            v = make_float4(__uint_as_float(t[4 * i]), __uint_as_float(t[4 * i + 1]), __uint_as_float(t[4 * i + 2]),
                            __uint_as_float(t[4 * i + 3]));
          *reinterpret_cast<float4*>(cluster_piece<BN>(part, row, half * (HW / 4) + j / 4 + i)) = v;
        }
      }
    }
  } else if constexpr (!TMA) {
    const int r0 = (warp - 10) * kLoadRows;  // of the stage's 256 rows: 128 of x, then 128 of w
    const RowWords<__nv_bfloat16> rows =
        r0 < kBM ? RowWords<__nv_bfloat16>(g.x, g.ldx, m0 + r0, g.M, g.K, lane)
                 : RowWords<__nv_bfloat16>(g.w, g.ldw, n0 + r0 - kBM, g.N, g.K, lane);
    uint8_t* const to = r0 < kBM ? sA + r0 * 128 : sB + (r0 - kBM) * 128;
    load_rows(
        rows, kb0, nkb, kBK,
        [&](int i) {
          return mbar_wait_warp(&empty[i % C::STAGES], ((i / C::STAGES) & 1) ^ 1, status, INL_DEV_TIMEOUT_PRODUCER);
        },
        [&](int i, int j, uint32_t word) {  // A_BYTES = B_BYTES here
          *reinterpret_cast<uint32_t*>(to + (i % C::STAGES) * C::A_BYTES + j * 128 + (((lane >> 2) ^ (j & 7)) << 4) +
                                       (lane & 3) * 4) = word;
        },
        [&](int i) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[i % C::STAGES]);
        });
  }
  tc_fence_before();
  cluster_sync_all();  // every partial tile is written
  if (warp >= 2 && warp < 10) cluster_finish<TO, BN, false>(g, part, threadIdx.x - 64, rank, S, m0, n0, wide != 0);
  cluster_sync_all();  // no CTA leaves while another may still read its partial tile
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMA ? 2 * BN : 4 * BN);
  }
}

template <typename TO, bool TMA>
cudaError_t launch_cluster(const CUtensorMap& ta, const CUtensorMap& tb, const LinearArgs& g, int S, int wide,
                           int* status, cudaStream_t s) {
  constexpr int BN = TMA ? 64 : 128;
  auto kern = linear_cluster_kernel<TO, TMA>;
  static std::atomic<unsigned long long> attr_set{0};
  const cudaError_t err = set_smem_limit_once(kern, ClusterCfg<BN>::SMEM_BYTES, attr_set);
  if (err != cudaSuccess) return err;
  const unsigned grid = ((g.M + kBM - 1) / kBM) * ((g.N + BN - 1) / BN) * S;
  return launch_cluster_pdl(kern, grid, threads_of(TMA), ClusterCfg<BN>::SMEM_BYTES, S, s, ta, tb, g, S, wide, status);
}

}  // namespace

cudaError_t linear_skinny(const LinearArgs& g, bool out_bf16, cudaStream_t s) {
  return out_bf16 ? launch_skinny_for<__nv_bfloat16>(g, s) : launch_skinny_for<float>(g, s);
}

cudaError_t linear_cluster(const LinearArgs& g, bool out_bf16, bool aligned, int S, int* status, cudaStream_t s) {
  auto pad8 = [](long long n) { return (n + 7) & ~7ll; };
  CUtensorMap ta = {}, tb = {};
  if (aligned && (!make_tma_2d_bf16(&ta, g.x, g.M, g.K, g.M == 1 ? pad8(g.K) : g.ldx, kBM, kBK) ||
                  !make_tma_2d_bf16(&tb, g.w, g.N, g.K, g.N == 1 ? pad8(g.K) : g.ldw, 64, kBK)))
    return cudaErrorInvalidValue;
  const int wide = linear_wide(g, out_bf16);
  auto run = [&](auto tma) {
    return out_bf16 ? launch_cluster<__nv_bfloat16, decltype(tma)::value>(ta, tb, g, S, wide, status, s)
                    : launch_cluster<float, decltype(tma)::value>(ta, tb, g, S, wide, status, s);
  };
  return aligned ? run(std::true_type()) : run(std::false_type());
}

}  // namespace inl
