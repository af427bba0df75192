// Linear layer with f32 operands on the tensor cores, to f32 accuracy.
//
// Each operand is split as x = hi + lo + (below 2^-21 |x|), hi its rounding to
// tf32 and lo the rest, which the tensor core reads as tf32, and the product is
// hi hi' + (hi lo' + lo hi') on tcgen05 kind::tf32 (lo lo' is below 2^-22 of the
// product). TMA brings f32 tiles; four warps move x's hi and lo into TMEM, where
// the products take their first operand from, two overwrite w's tile with its hi
// and write lo beside. The tensor core's f32 accumulator truncates, which over a
// long K costs more than the split does (a sum of 4096 bf16 products was off by
// 4.4e-6, toward zero), so the two kinds of product have accumulators of their
// own, and the large one is moved out and summed in registers, rounded to
// nearest, every 128 of K; the small one is 2^-11 of it and stays.
//
// A CTA walks over 128 x 128 tiles, or a cluster of S CTAs shares out the K of
// one, as in linear_cluster_kernel. A sum that comes out NaN is computed again as
// a plain f32 sum: the split turns an infinite (or rounding to infinity) operand
// into inf - inf, and a row that holds one must still give what f32 gives. One lane
// computes it, 0.14 us per element of K: 1024 x 1024 x 1024 with an infinity in every
// row 4.7 ms, 1024 x 4736 x 320000 5 s, which is why waits behind it end only when
// it stands still (wait_alive).
//
// 1024 x 4096 x 1024: 56 us = 154 TFLOP/s of f32, off by 3.5e-7 (an f32 library
// product: 162 us, off by 5.7e-7); 8192 x 4096 x 4096: 1.35 ms = 203 TFLOP/s,
// where the products alone, the splitting left out, take 1.19 ms at the clock
// that the power limit leaves. With both operands split in shared memory, 72 us
// on the first: the tile's 224 KB of shared memory traffic a K block bound it; one
// tile to a CTA 62 us. Rows of odd strides: 97 us.
#include <algorithm>
#include <type_traits>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "kernels.h"
#include "linear.h"

namespace inl {

namespace {

constexpr int kBM = 128, kBN = 128, kBK = 32;  // 32 f32: one 128-byte swizzle row
constexpr int kTile = kBM * kBK * 4;            // one operand's f32 tile
constexpr int kChunk = 4;                       // K blocks between promotions of the large sum
constexpr int kSplitX = 4, kSplitW = 2;         // splitting warps
// The ring in shared memory. TMA: 4 stages of x as loaded (its hi and lo go to
// TMEM), w hi (in place of the loaded w) and w lo; then 4 KB for each sum warp to
// store through. Else: 3 stages of x hi, w hi, x lo, w lo.
constexpr int kStagesTma = 4, kStagesOdd = 3, kRing = 12 * kTile;
static_assert(kStagesTma * 3 * kTile == kRing && kStagesOdd * 4 * kTile == kRing, "ring");
constexpr int kSmem = kRing + 8 * 4096 + 1024 + 256;
// TMEM: two large accumulators and the small one, 128 columns each; then, TMA:
// two buffers of x hi and x lo, 32 columns each; else a total.
constexpr int kTmemCols = 512;

// Instruction descriptor of kind::tf32: D f32, A and B tf32, both K-major.
__host__ __device__ constexpr uint32_t idesc_tf32(int M, int N) {
  return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// The same with A in TMEM (row = lane, k = column).
__device__ __forceinline__ void umma_tf32_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
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
constexpr int threads_of(bool tma) { return 320 + 32 * (tma ? kSplitX + kSplitW : kLoadWarps); }

// Phase bookkeeping of a ring of n slots: its i-th use is slot i % n, and the
// waits on that use are for parity (i / n) & 1.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) slot = 0, phase ^= 1;
  }
};

// S CTAs (a cluster) share out the K of one tile; with S = 1 and TMA, a CTA walks
// over tiles, and a tile's epilogue runs under the next one's products.
template <typename TO, bool TMA>
__global__ void __launch_bounds__(threads_of(TMA), 1)
    linear_f32_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, LinearArgs g,
                      int S, int wide, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const stage_out = smem + kRing;
  constexpr int kStages = TMA ? kStagesTma : kStagesOdd, kStageBytes = kRing / kStages;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + 8 * 4096);  // f32 tiles landed
  uint64_t* split = full + kStages;                                    // hi and lo written
  uint64_t* empty = split + kStages;                                   // ... products done
  uint64_t* xfree = empty + kStages;                                   // ... those that read x from TMEM buffer b
  uint64_t* tfull = xfree + 2;                                         // large accumulator a complete
  uint64_t* tempty = tfull + 2;                                        // ... moved out
  uint64_t* sempty = tempty + 2;                                       // small accumulator moved out
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sempty + 1);

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int n_tiles = (g.N + kBN - 1) / kBN;
  const bool walk = TMA && S == 1;
  const int first = blockIdx.x / S;
  const int end = walk ? (g.M + kBM - 1) / kBM * n_tiles : first + 1, stride = gridDim.x;
  const int k_blocks = (g.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<long long>(k_blocks) * rank / S);
  const int nkb = static_cast<int>(static_cast<long long>(k_blocks) * (rank + 1) / S) - kb0;  // > 0: S <= k_blocks
  const int chunks = (nkb + kChunk - 1) / kChunk;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&split[s], TMA ? kSplitX + kSplitW : kLoadWarps);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 8);
      mbar_init(&xfree[a], 1);
    }
    mbar_init(sempty, 8);
    if (TMA) *redo_beat() = 0;
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

  // CTAs that walk over tiles compute NaNs again under the next tile's products: every wait may be behind that
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return TMA ? wait_alive(bar, parity, status, code) : mbar_wait(bar, parity, status, code);
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity, int code) {
    return __all_sync(0xffffffffu, wait(bar, parity, code));
  };

  if (warp == 0) {
    if (TMA && lane == 0) {
      Ring in;
      int issued = 0;  // at most kStages matter
      bool ok = true;
      for (int tile = first; tile < end && ok; tile += stride) {
        const int m0 = tile / n_tiles * kBM, n0 = tile % n_tiles * kBN;
        for (int i = 0; i < nkb; ++i, in.next(kStages)) {
          if (!(ok = wait(&empty[in.slot], in.phase ^ 1, INL_DEV_TIMEOUT_PRODUCER))) break;
          uint8_t* base = smem + in.slot * kStageBytes;
          mbar_expect_tx(&full[in.slot], 2 * kTile);
          tma_load_2d(base, &tmA, &full[in.slot], (kb0 + i) * kBK, m0);
          tma_load_2d(base + kTile, &tmB, &full[in.slot], (kb0 + i) * kBK, n0);
          issued = min(issued + 1, kStages);
        }
      }
      // every copy has landed before the CTA can leave: the last `issued` uses
      for (int f = issued; f > 0; --f) {
        const int back = in.slot - f;  // slots before in.slot are in this phase, the others in the one before
        const int slot = back < 0 ? back + kStages : back;
        if (!wait(&full[slot], back < 0 ? in.phase ^ 1 : in.phase, INL_DEV_TIMEOUT_DRAIN)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_tf32(kBM, kBN);
      const uint32_t small = tmem + 2 * kBN;
      Ring out, x, acc;
      uint32_t tile_phase = 0;
      bool ok = true;
      for (int tile = first; tile < end && ok; tile += stride, tile_phase ^= 1) {
        if (!(ok = wait(sempty, tile_phase ^ 1, INL_DEV_TIMEOUT_MMA))) break;
        for (int i = 0; i < nkb; ++i, out.next(kStages), x.next(2)) {
          if (i % kChunk == 0 &&
              !(ok = wait(&tempty[acc.slot], acc.phase ^ 1, INL_DEV_TIMEOUT_MMA)))
            break;
          if (!(ok = wait(&split[out.slot], out.phase, INL_DEV_TIMEOUT_MMA))) break;
          tc_fence_after();
          // a stage: x, w hi, w lo (TMA); x hi, w hi, x lo, w lo
          const uint64_t st = sw128_kmajor_desc(smem_u32(smem + out.slot * kStageBytes)), wh = st + (kTile >> 4);
          const uint64_t wl = st + ((TMA ? 2 : 3) * kTile >> 4), xl = st + (2 * kTile >> 4);
          const uint32_t xt = tmem + 3 * kBN + x.slot * 2 * kBK;
          const uint32_t big = tmem + acc.slot * kBN;
#pragma unroll
          for (int kk = 0; kk < kBK / 8; ++kk) {  // 8 of K: 32 bytes of each row
            const uint64_t o = static_cast<uint64_t>(kk * 2);
            const uint32_t more = i % kChunk != 0 || kk != 0, any = i != 0 || kk != 0;
            if constexpr (TMA) {
              umma_tf32_ts(big, xt + kk * 8, wh + o, idesc, more);
              umma_tf32_ts(small, xt + kk * 8, wl + o, idesc, any);
              umma_tf32_ts(small, xt + kBK + kk * 8, wh + o, idesc, 1u);
            } else {
              umma_tf32(big, st + o, wh + o, idesc, more);
              umma_tf32(small, st + o, wl + o, idesc, any);
              umma_tf32(small, xl + o, wh + o, idesc, 1u);
            }
          }
          umma_commit(&empty[out.slot]);
          if (TMA) umma_commit(&xfree[x.slot]);
          if (i % kChunk == kChunk - 1 || i == nkb - 1) {
            umma_commit(&tfull[acc.slot]);
            acc.next(2);
          }
        }
      }
    }
  } else if (warp < 10) {
    // thread = tile row (lane quadrant warp % 4), 64 columns. Sums in registers;
    // in TMEM beside the loading warps, whose loads need them.
    const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 64;
    const uint32_t t_total = t_row + 3 * kBN;
    constexpr int R = TMA ? 64 : 16;
    float sum[R];
    Ring acc;
    bool ok = true;
    for (int tile = first; tile < end; tile += stride) {
#pragma unroll
      for (int j = 0; j < R; ++j) sum[j] = 0.f;
      for (int c = 0; c < chunks; ++c, acc.next(2)) {
        if (!(ok = wait_warp(&tfull[acc.slot], acc.phase, INL_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < 64; j += 16) {
          if constexpr (TMA) {
            uint32_t r[16];
            tmem_ld16(t_row + acc.slot * kBN + j, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[j + i] += __uint_as_float(r[i]);
          } else {
            tmem_add16(t_total + j, t_row + acc.slot * kBN + j, c == 0);
          }
        }
        if constexpr (!TMA) tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc.slot]);
      }
      if (!ok) break;
      // the last products are done: the small sum, and, in a cluster, the
      // partial tile, which the ring's memory takes
#pragma unroll
      for (int j = 0; j < 64; j += 16) {
        uint32_t r[16], t[16];
        tmem_ld16(t_row + 2 * kBN + j, r);
        if constexpr (!TMA) tmem_ld16(t_total + j, t);
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) + (TMA ? sum[(j + i) % R] : __uint_as_float(t[i]));
        if (walk) {
          if constexpr (TMA) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[j + i] = v[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(cluster_piece<kBN>(smem, row, half * 16 + j / 4 + i)) =
                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
      }
      if constexpr (TMA) {
        if (walk) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty);
          const int m = tile / n_tiles * kBM + quad * 32, n = tile % n_tiles * kBN + half * 64;
          if (m < g.M && n < g.N) {
            warp_finish32<TO, true>(g, stage_out + (warp - 2) * 4096, sum, m, n, lane, wide != 0);
            if (n + 32 < g.N) warp_finish32<TO, true>(g, stage_out + (warp - 2) * 4096, sum + 32, m, n + 32, lane, wide != 0);
          }
        }
      }
    }
  } else if constexpr (!TMA) {
    const int m0 = first / n_tiles * kBM, n0 = first % n_tiles * kBN;
    const int r0 = (warp - 10) * kLoadRows;  // of the stage's 256 rows: 128 of x, then 128 of w
    const RowWords<float> rows = r0 < kBM ? RowWords<float>(g.x, g.ldx, m0 + r0, g.M, g.K, lane)
                                          : RowWords<float>(g.w, g.ldw, n0 + r0 - kBM, g.N, g.K, lane);
    load_rows(
        rows, kb0, nkb, kBK,
        [&](int i) {
          return wait_warp(&empty[i % kStages], ((i / kStages) & 1) ^ 1, INL_DEV_TIMEOUT_PRODUCER);
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
    Ring in, x;
    bool ok = true;
    const int row = (warp & 3) * 32 + lane, tid = threadIdx.x - 32 * (10 + kSplitX);
    const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 3 * kBN;
    for (int tile = first; tile < end && ok; tile += stride) {
      for (int i = 0; i < nkb; ++i, in.next(kStages), x.next(2)) {
        const bool of_x = warp < 10 + kSplitX;
        if (of_x && !(ok = wait_warp(&xfree[x.slot], x.phase ^ 1, INL_DEV_TIMEOUT_PRODUCER))) break;
        if (!(ok = wait_warp(&full[in.slot], in.phase, INL_DEV_TIMEOUT_PRODUCER))) break;
        uint8_t* const at = smem + in.slot * kStageBytes;
        if (of_x) {
          // x: thread = row (lane quadrant warp % 4), from shared memory to TMEM
          tc_fence_after();
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(at + row * 128 + ((j ^ (row & 7)) << 4));
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float h = tf32_of(e[k]);
              hi[4 * j + k] = __float_as_uint(h);
              lo[4 * j + k] = __float_as_uint(e[k] - h);
            }
          }
          tmem_st32(t_row + x.slot * 2 * kBK, hi);
          tmem_st32(t_row + x.slot * 2 * kBK + kBK, lo);
          tmem_st_wait();
          tc_fence_before();
        } else {
          // w: hi in place, lo beside (offsets from one base: the compiler sees
          // that the loads ahead do not meet the stores)
          uint8_t* const base = at + kTile + tid * 16;
#pragma unroll
          for (int o = 0; o < kTile; o += 32 * kSplitW * 16) {
            const float4 v = *reinterpret_cast<const float4*>(base + o);
            const float4 h = make_float4(tf32_of(v.x), tf32_of(v.y), tf32_of(v.z), tf32_of(v.w));
            *reinterpret_cast<float4*>(base + o) = h;
            *reinterpret_cast<float4*>(base + o + kTile) = make_float4(v.x - h.x, v.y - h.y, v.z - h.z, v.w - h.w);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&split[in.slot]);
      }
    }
  }
  tc_fence_before();
  cluster_sync_all();  // every partial tile is written
  if (!walk && warp >= 2 && warp < 10)
    cluster_finish<TO, kBN, true>(g, smem, threadIdx.x - 64, rank, S, first / n_tiles * kBM, first % n_tiles * kBN,
                                  wide != 0);
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
  int grid = ((g.M + kBM - 1) / kBM) * ((g.N + kBN - 1) / kBN) * S;
  if (TMA && S == 1) grid = std::min(grid, num_sms_cached());
  return launch_cluster_pdl(kern, static_cast<unsigned>(grid), threads_of(TMA), kSmem, S, s, ta, tb, g, S, wide, status);
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
