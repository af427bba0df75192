// Linear layer with f32 operands on the tensor cores, to f32 accuracy.
//
// Each operand is split as x = hi + lo + (below 2^-23 |x|), hi and lo its tf32
// roundings, and the product is hi hi' + (hi lo' + lo hi') on tcgen05 kind::tf32
// (lo lo' is below 2^-22 of the product). The split happens in shared memory:
// TMA brings f32 tiles, four warps overwrite them with hi and write lo beside.
// The tensor core's f32 accumulator truncates, which over a long K costs more
// than the split does (a sum of 4096 bf16 products was off by 4.4e-6, toward
// zero), so the two kinds of product have accumulators of their own, and the
// large one is moved out and summed in registers, rounded to nearest, every 128
// of K; the small one is 2^-11 of it and stays.
//
// One 128 x 128 tile per cluster of S CTAs, which share out K as in
// linear_cluster_kernel. A sum that comes out NaN is computed again as a plain
// f32 sum: the split turns an infinite (or rounding to infinity) operand into
// inf - inf, and a row that holds one must still give what f32 gives.
//
// Bound by shared memory: a 128 x 128 x 32 block writes 32 KB (TMA), reads it,
// writes 64 KB (hi, lo) and is read by 12 products of 8 KB, 224 KB or 1750 cycles
// of the SM's 128 bytes a cycle, against 768 cycles of products. 1024 x 4096 x
// 1024: 72 us = 120 TFLOP/s of f32 (an f32 library product: 162 us, off by
// 5.7e-7 where this is off by 3.5e-7); 8192 x 1024 x 4096: 444 us; rows of odd
// strides 92 and 561 us. With hi left to the tensor core's own truncation of
// what TMA wrote 63 us, but an error of 6.3e-7, all of it toward zero.
#include <type_traits>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "kernels.h"
#include "linear.h"

namespace inl {

namespace {

constexpr int kBM = 128, kBN = 128, kBK = 32;  // 32 f32: one 128-byte swizzle row
constexpr int kStages = 3;
constexpr int kTile = kBM * kBK * 4;    // one operand's f32 tile
constexpr int kStageBytes = 4 * kTile;  // x hi, w hi (in place of the loaded f32), x lo, w lo
constexpr int kChunk = 4;               // K blocks between promotions of the large sum
constexpr int kConvWarps = 4;
constexpr int kSmem = kStages * kStageBytes + 1024 + 256;
constexpr int kTmemCols = 512;  // two large accumulators, the small one and a total, 128 columns each

// Instruction descriptor of kind::tf32: D f32, A and B tf32, both K-major.
__host__ __device__ constexpr uint32_t idesc_tf32(int M, int N) {
  return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void umma_tf32(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// x rounded to tf32's 10 fraction bits, ties away from zero. An infinity stays one; a NaN may not (its difference
// from this does).
__device__ __forceinline__ float tf32_of(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}

// TMA, MMA, 8 sum warps, the splitting warps; or, for rows that no TMA map
// takes, sixteen warps that load them word by word and split them on the way.
constexpr int threads_of(bool tma) { return 320 + 32 * (tma ? kConvWarps : kLoadWarps); }

template <typename TO, bool TMA>
__global__ void __launch_bounds__(threads_of(TMA), 1)
    linear_f32_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, LinearArgs g,
                      int S, int wide, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);  // f32 tiles landed
  uint64_t* split = full + kStages;                                            // hi and lo written
  uint64_t* empty = split + kStages;                                           // products done
  uint64_t* tfull = empty + kStages;                                           // large accumulator a complete
  uint64_t* tempty = tfull + 2;                                                // ... moved out
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / S;
  const int n_tiles = (g.N + kBN - 1) / kBN;
  const int m0 = tile / n_tiles * kBM, n0 = tile % n_tiles * kBN;
  const int k_blocks = (g.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<long long>(k_blocks) * rank / S);
  const int nkb = static_cast<int>(static_cast<long long>(k_blocks) * (rank + 1) / S) - kb0;  // > 0: S <= k_blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&split[s], TMA ? kConvWarps : kLoadWarps);
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
    tmem_alloc(tmem_holder, kTmemCols);
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
        const int st = issued % kStages;
        uint8_t* base = smem + st * kStageBytes;
        if (!mbar_wait(&empty[st], ((issued / kStages) & 1) ^ 1, status, INL_DEV_TIMEOUT_PRODUCER)) break;
        mbar_expect_tx(&full[st], 2 * kTile);
        tma_load_2d(base, &tmA, &full[st], (kb0 + issued) * kBK, m0);
        tma_load_2d(base + kTile, &tmB, &full[st], (kb0 + issued) * kBK, n0);
      }
      for (int f = max(0, issued - kStages); f < issued; ++f)  // every copy has landed before the CTA can leave
        if (!mbar_wait(&full[f % kStages], (f / kStages) & 1, status, INL_DEV_TIMEOUT_DRAIN)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_tf32(kBM, kBN);
      const uint32_t small = tmem + 2 * kBN;
      for (int i = 0; i < nkb; ++i) {
        const int st = i % kStages, chunk = i / kChunk, acc = chunk & 1;
        if (i % kChunk == 0 && !mbar_wait(&tempty[acc], ((chunk >> 1) & 1) ^ 1, status, INL_DEV_TIMEOUT_MMA)) break;
        if (!mbar_wait(&split[st], (i / kStages) & 1, status, INL_DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint64_t xh = sw128_kmajor_desc(smem_u32(smem + st * kStageBytes)), wh = xh + (kTile >> 4);
        const uint64_t xl = xh + (2 * kTile >> 4), wl = xh + (3 * kTile >> 4);
        const uint32_t big = tmem + acc * kBN;
#pragma unroll
        for (int kk = 0; kk < kBK / 8; ++kk) {  // 8 of K: 32 bytes of each row
          const uint64_t o = static_cast<uint64_t>(kk * 2);
          umma_tf32(big, xh + o, wh + o, idesc, (i % kChunk != 0 || kk != 0) ? 1u : 0u);
          umma_tf32(small, xh + o, wl + o, idesc, (i != 0 || kk != 0) ? 1u : 0u);
          umma_tf32(small, xl + o, wh + o, idesc, 1u);
        }
        umma_commit(&empty[st]);
        if (i % kChunk == kChunk - 1 || i == nkb - 1) umma_commit(&tfull[acc]);
      }
    }
  } else if (warp < 10) {
    // thread = tile row (lane quadrant warp % 4), 64 columns
    const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 64;
    const int chunks = (nkb + kChunk - 1) / kChunk;
    // Sums in registers; in TMEM beside the loading warps, whose loads need them.
    constexpr int R = TMA ? 64 : 16;
    const uint32_t t_total = t_row + 3 * kBN;
    float sum[R];
#pragma unroll
    for (int j = 0; j < R; ++j) sum[j] = 0.f;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const int acc = c & 1;
      if (!(ok = mbar_wait_warp(&tfull[acc], (c >> 1) & 1, status, INL_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < 64; j += 16) {
        if constexpr (TMA) {
          uint32_t r[16];
          tmem_ld16(t_row + acc * kBN + j, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[j + i] += __uint_as_float(r[i]);
        } else {
          tmem_add16(t_total + j, t_row + acc * kBN + j, c == 0);
        }
      }
      if constexpr (!TMA) tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
    if (ok) {
      // every product is done, so the ring's memory takes the partial tile
#pragma unroll
      for (int j = 0; j < 64; j += 16) {
        uint32_t r[16], t[16];
        tmem_ld16(t_row + 2 * kBN + j, r);
        if constexpr (!TMA) tmem_ld16(t_total + j, t);
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) + (TMA ? sum[(j + i) % R] : __uint_as_float(t[i]));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(cluster_piece<kBN>(smem, row, half * 16 + j / 4 + i)) =
              make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    }
  } else if constexpr (!TMA) {
    const int r0 = (warp - 10) * kLoadRows;  // of the stage's 256 rows: 128 of x, then 128 of w
    const RowWords<float> rows = r0 < kBM ? RowWords<float>(g.x, g.ldx, m0 + r0, g.M, g.K, lane)
                                          : RowWords<float>(g.w, g.ldw, n0 + r0 - kBM, g.N, g.K, lane);
    load_rows(
        rows, kb0, nkb, kBK,
        [&](int i) {
          return mbar_wait_warp(&empty[i % kStages], ((i / kStages) & 1) ^ 1, status, INL_DEV_TIMEOUT_PRODUCER);
        },
        [&](int i, int j, uint32_t word) {
          const float v = __uint_as_float(word), h = tf32_of(v);
          float* to = reinterpret_cast<float*>(smem + (i % kStages) * kStageBytes + (r0 + j) * 128 +
                                               (((lane >> 2) ^ (j & 7)) << 4) + (lane & 3) * 4);
          to[0] = h;
          to[2 * kTile / 4] = v - h;
        },
        [&](int i) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&split[i % kStages]);
        });
  } else {
    const int tid = threadIdx.x - 320;
    for (int i = 0; i < nkb; ++i) {
      const int st = i % kStages;
      if (!mbar_wait_warp(&full[st], (i / kStages) & 1, status, INL_DEV_TIMEOUT_PRODUCER)) break;
      uint8_t* base = smem + st * kStageBytes + tid * 16;
#pragma unroll 8
      for (int o = 0; o < 2 * kTile; o += 32 * kConvWarps * 16) {
        const float4 v = *reinterpret_cast<const float4*>(base + o);
        const float4 h = make_float4(tf32_of(v.x), tf32_of(v.y), tf32_of(v.z), tf32_of(v.w));
        *reinterpret_cast<float4*>(base + o) = h;
        *reinterpret_cast<float4*>(base + o + 2 * kTile) =
            make_float4(v.x - h.x, v.y - h.y, v.z - h.z, v.w - h.w);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&split[st]);
    }
  }
  tc_fence_before();
  cluster_sync_all();  // every partial tile is written
  if (warp >= 2 && warp < 10)
    cluster_finish<TO, kBN, true>(g, smem, threadIdx.x - 64, rank, S, m0, n0, wide != 0);
  cluster_sync_all();  // no CTA leaves while another may still read its partial tile
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename TO, bool TMA>
cudaError_t launch_f32(const CUtensorMap& ta, const CUtensorMap& tb, const LinearArgs& g, int S, int wide, int* status,
                       cudaStream_t s) {
  auto kern = linear_f32_kernel<TO, TMA>;
  static std::atomic<unsigned long long> attr_set{0};
  const cudaError_t err = set_smem_limit_once(kern, kSmem, attr_set);
  if (err != cudaSuccess) return err;
  const unsigned grid = ((g.M + kBM - 1) / kBM) * ((g.N + kBN - 1) / kBN) * S;
  return launch_cluster_pdl(kern, grid, threads_of(TMA), kSmem, S, s, ta, tb, g, S, wide, status);
}

}  // namespace

bool linear_f32_takes(const LinearArgs& g) {
  auto rows_ok = [](const void* p, long long ld, long long rows) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || (ld % 4 == 0 && ld * 4 < (1ll << 40)));
  };
  return g.K > 0 && rows_ok(g.x, g.ldx, g.M) && rows_ok(g.w, g.ldw, g.N);
}

cudaError_t linear_f32(const LinearArgs& g, bool out_bf16, bool aligned, int S, int* status, cudaStream_t s) {
  auto pad4 = [](long long n) { return (n + 3) & ~3ll; };
  CUtensorMap ta = {}, tb = {};
  if (aligned && (!make_tma_2d_f32(&ta, g.x, g.M, g.K, g.M == 1 ? pad4(g.K) : g.ldx, kBM, kBK) ||
                  !make_tma_2d_f32(&tb, g.w, g.N, g.K, g.N == 1 ? pad4(g.K) : g.ldw, kBN, kBK)))
    return cudaErrorInvalidValue;
  const int wide = linear_wide(g, out_bf16);
  auto run = [&](auto tma) {
    return out_bf16 ? launch_f32<__nv_bfloat16, decltype(tma)::value>(ta, tb, g, S, wide, status, s)
                    : launch_f32<float, decltype(tma)::value>(ta, tb, g, S, wide, status, s);
  };
  return aligned ? run(std::true_type()) : run(std::false_type());
}

}  // namespace inl
