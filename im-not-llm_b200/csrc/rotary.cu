// Rotary positions, alone and behind the per-head norms of queries and keys,
// over packed token rows: inl_cuda_rope, inl_cuda_qk_norm_rotary and the host's
// inl_cuda_rope_frequencies.
//
//   pair (a, b) of a head -> scale (a cos t - b sin t, b cos t + a sin t),
//   t = pos[token] * inv_freq[pair]
//
// The angle is formed in 64 bits and reduced to within an eighth of a turn
// before it becomes 32 bits: at position 10^6 a 32-bit product would be off by
// up to 0.03 radians, the reduced one is off by 3e-8.
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <type_traits>
#include <vector>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "hook_checks.h"
#include "kernels.h"
#include "turns.h"

namespace inl {

namespace {

enum RotaryNorm : int { kNoNorm = 0, kRms = 1, kLayer = 2 };

// One set of heads (queries, or keys): rows of `heads` heads, in and out.
struct HeadSet {
  const void* x;
  void* out;
  const float* w;
  const float* b;
  long long ldx, hsx, ldo;
  int heads;
};

struct RotaryArgs {
  HeadSet set[2];
  int T, d, rot, interleaved;
  float eps, scale, sin_sign;
  const int* pos;
  const double* inv_freq;
};

// Any head width, stride and alignment: a warp per (token, head), a lane per
// pair (and per feature that is copied), so that in-place rows are read and
// written by one lane alone. Two passes over the head when it is normed. 65536
// tokens of 24 bf16 heads of 128 at an odd stride: 505 us, RMS-normed 751, bound by
// angles formed anew for each head and 2-byte accesses.
template <typename T, int NORM>
__global__ void __launch_bounds__(256) rotary_any_kernel(RotaryArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.set[0].heads + a.set[1].heads;
  const long long items = static_cast<long long>(a.T) * heads;
  const long long step = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long item = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items;
       item += step) {
    const long long t = item / heads;
    int h = static_cast<int>(item - t * heads);
    const bool second = h >= a.set[0].heads;
    const HeadSet& st = a.set[second];
    if (second) h -= a.set[0].heads;
    const T* x = static_cast<const T*>(st.x) + t * st.ldx + h * st.hsx;
    T* out = static_cast<T*>(st.out) + t * st.ldo + static_cast<long long>(h) * a.d;
    float mean = 0.f, inv = 1.f;
    if constexpr (NORM != kNoNorm) {
      if constexpr (NORM == kLayer) {
        float sum = 0.f;
        for (int j = lane; j < a.d; j += 32) sum += load_f(x + j);
        mean = warp_sum(sum) / static_cast<float>(a.d);
      }
      float ss = 0.f;
      for (int j = lane; j < a.d; j += 32) {
        const float v = load_f(x + j) - mean;
        ss = fmaf(v, v, ss);
      }
      inv = rsqrtf(warp_sum(ss) / static_cast<float>(a.d) + a.eps);
    }
    auto value = [&](int j) {
      float v = load_f(x + j);
      if constexpr (NORM != kNoNorm) {
        v = (v - mean) * inv;
        if (st.w) v *= st.w[j];
        if constexpr (NORM == kLayer)
          if (st.b) v += st.b[j];
      }
      return v;
    };
    const int half = a.rot / 2;
    const int pos = half ? a.pos[t] : 0;
    for (int i = lane; i < half; i += 32) {
      const int ja = a.interleaved ? 2 * i : i, jb = a.interleaved ? 2 * i + 1 : i + half;
      float c, s;
      turn_of(pos, turn_step(a.inv_freq[i]), c, s);
      c *= a.scale;
      s *= a.scale * a.sin_sign;
      const float va = value(ja), vb = value(jb);
      store_f(out + ja, va * c - vb * s);
      store_f(out + jb, vb * c + va * s);
    }
    for (int j = a.rot + lane; j < a.d; j += 32) store_f(out + j, value(j));
  }
}

template <typename T, int NORM>
cudaError_t launch_any(const RotaryArgs& a, cudaStream_t s) {
  const long long items = static_cast<long long>(a.T) * (a.set[0].heads + a.set[1].heads);
  const long long blocks = std::min<long long>((items + 7) / 8, 1 << 20);
  return launch_plain(rotary_any_kernel<T, NORM>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a);
}

// E consecutive values in one access.
template <typename T, int E>
struct Vec {
  static constexpr int BYTES = E * static_cast<int>(sizeof(T));
  using Raw = std::conditional_t<BYTES == 16, uint4, std::conditional_t<BYTES == 8, uint2, uint32_t>>;
  static __device__ __forceinline__ void unpack(const Raw& r, float* v) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const float2 f = unpack_bf16x2(u[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[i] = __uint_as_float(u[i]);
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float* v) {
    Raw r;
    uint32_t* u = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) {
      if constexpr (sizeof(T) == 2) u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else u[i] = __float_as_uint(v[i]);
    }
    return r;
  }
};

// The bandwidth-bound form. A head is cut into units of two E-vectors: E pairs
// of the rotation (vectors i E and half + i E of the half layout, 2 E
// consecutive features of the interleaved one) or 2 E features that are
// copied, one unit to a lane, 2^log_lanes lanes to a head. So a lane turns its
// own registers, without an exchange, and in place writes what it read. A warp
// takes 2^log_tokens tokens at a time (one, where the heads are many), gives
// each as many lane groups, and a group takes every step-th head of its token,
// or of its run of heads (blockIdx.y: some, where the tokens are few). The
// warp computes its tokens' cos and sin once, into shared memory of its own, so
// no warp waits for another. A lane asks for a head of the next batch (of KI
// heads, or of the next tokens) as soon as it has taken this one out of the
// registers.
//
// Bound by memory: 65536 tokens of 24 bf16 heads of 128, rotated 123 us = 6.5
// TB/s (all of a copy's rate; 126 over a second of them, at the power limit),
// RMS-normed and rotated 140 us = 5.7 TB/s (148), with LayerNorm 167 (174); 20011
// f32 tokens of 12 heads of 64, interleaved, 25 us = 5.0 TB/s. Tried on the first
// of these (us): a block per 4 tokens, a barrier between its cos / sin and its
// heads 175; blocks that walk over tiles, with that barrier 153 to 178; 2 / 4
// heads in flight 137 / 187 (registers); 8-byte vectors 202; more resident
// warps at fewer registers 149 and more; two features to an instruction 125
// (normed 143); a head's address made anew for each load 124 (normed 145).
template <typename T, int E, int NORM, bool INTER, int KI>
__global__ void __launch_bounds__(256, 2) rotary_vec_kernel(RotaryArgs a, int log_lanes, int log_tokens, int run) {
  using V = Vec<T, E>;
  using Raw = typename V::Raw;
  constexpr int Q = E / 2;          // float4s of a unit's cos and sin, or of its weights
  extern __shared__ float4 smem4[];  // per warp [tokens][Q][pair units] (cos, sin, cos, sin); [q, k][w, b][Q][units]; steps
  const int half = a.rot / 2, heads = a.set[0].heads + a.set[1].heads, hq = a.set[0].heads;
  const int warp = threadIdx.x >> 5, wl = threadIdx.x & 31;
  const int lane = wl & ((1 << log_lanes) - 1), group = wl >> log_lanes;
  const int log_step = 5 - log_lanes - log_tokens, step = 1 << log_step;
  const int pair_units = half / E, units = a.d / (2 * E);
  const bool active = lane < units, turned = lane < pair_units;
  auto first_of = [&](int u) { return u >= pair_units ? a.rot + 2 * E * (u - pair_units) : INTER ? 2 * E * u : E * u; };
  const int f = active ? first_of(lane) : 0;
  const int gap = turned && !INTER ? half : E;  // from a lane's first vector to its second
  const int tok = group >> log_step;
  const int run0 = blockIdx.y * run, run1 = min(run0 + run, heads);  // this block's heads
  const int h0 = run0 + (group & (step - 1));
  const int tiles = (a.T - 1) / (1 << log_tokens) + 1;  // of 2^log_tokens tokens
  const int cs_n = half / 2 << log_tokens;              // float4s of a warp's cos and sin
  float4* const cs = smem4 + warp * cs_n;
  float4* const wsm = smem4 + 8 * cs_n;
  uint64_t* const steps = reinterpret_cast<uint64_t*>(wsm + (NORM == kNoNorm ? 0 : a.d));  // [half]

  // A row's q heads and k heads, at this lane's features; the keys' pointer is
  // set back by hq heads, so that head h of either lies h strides on.
  const int hs_q = static_cast<int>(a.set[0].hsx), hs_k = static_cast<int>(a.set[1].hsx);
  auto row_at = [&](int tile, const T*& q, const T*& k) {
    const long long row = min((tile << log_tokens) + tok, a.T - 1);
    q = static_cast<const T*>(a.set[0].x) + row * a.set[0].ldx + f;
    k = static_cast<const T*>(a.set[1].x) + row * a.set[1].ldx + (f - hq * hs_k);
  };
  auto load = [&](const T* q, const T* k, int h, Raw (&raw)[2]) {
    h = min(h, run1 - 1);
    const bool second = h >= hq;
    const T* x = (second ? k : q) + h * (second ? hs_k : hs_q);
    raw[0] = *reinterpret_cast<const Raw*>(x);
    raw[1] = *reinterpret_cast<const Raw*>(x + gap);
  };
  const int turns = half << log_tokens;
  // lane t: the position of the warp's token t
  auto load_pos = [&](int tile) {
    return half && wl < 1 << log_tokens ? a.pos[min((tile << log_tokens) + wl, a.T - 1)] : 0;
  };

  int tile = blockIdx.x * 8 + warp;
  const int tile_step = gridDim.x * 8;
  Raw raw[KI][2];
  int pos = 0;
  const T *xq = nullptr, *xk = nullptr;
  if (tile < tiles) {
    row_at(tile, xq, xk);
#pragma unroll
    for (int k = 0; k < KI; ++k) load(xq, xk, h0 + k * step, raw[k]);
    pos = load_pos(tile);
  }
  for (int i = threadIdx.x; i < half; i += 256) steps[i] = turn_step(a.inv_freq[i]);
  if constexpr (NORM != kNoNorm) {
    float* const wf = reinterpret_cast<float*>(wsm);
    for (int i = threadIdx.x; i < 2 * units * 2 * E; i += 256) {
      const int k = i / (units * 2 * E), u = i / (2 * E) % units, e = i % (2 * E);
      const int ff = first_of(u) + (e < E ? e : (u < pair_units && !INTER ? half : E) + e - E);
      const HeadSet& st = a.set[k];
      float* to = wf + ((2 * k * Q + e / 4) * units + u) * 4 + e % 4;
      *to = st.w ? st.w[ff] : 1.f;
      if constexpr (NORM == kLayer) to[4 * Q * units] = st.b ? st.b[ff] : 0.f;
    }
  }
  __syncthreads();

  for (; tile < tiles; tile += tile_step) {
    const int next = tile + tile_step;
    __syncwarp();  // the last tokens' cos and sin have been read
#pragma unroll 2
    for (int i = wl; i < (turns + 31 & ~31); i += 32) {  // whole warps: the shuffle
      const int t = log_tokens ? min(i / half, (1 << log_tokens) - 1) : 0, p = i - t * half;
      const int at = __shfl_sync(0xffffffffu, pos, t);
      if (i < turns) {
        float co, si;
        turn_of(at, steps[p], co, si);
        reinterpret_cast<float2*>(cs)[t * half + (p % E / 2 * pair_units + p / E) * 2 + (p & 1)] =
            make_float2(co * a.scale, si * (a.scale * a.sin_sign));
      }
    }
    const T *nq = xq, *nk = xk;
    if (next < tiles) {
      pos = load_pos(next);
      row_at(next, nq, nk);
    }
    __syncwarp();
    float c[E], sn[E];
    if (turned) {
#pragma unroll
      for (int j = 0; j < Q; ++j) {
        const float4 r = cs[(tok * Q + j) * pair_units + lane];
        c[2 * j] = r.x, sn[2 * j] = r.y, c[2 * j + 1] = r.z, sn[2 * j + 1] = r.w;
      }
    }
    const long long row = (tile << log_tokens) + tok;
    const bool mine = active && row < a.T;
    T* const oq = static_cast<T*>(a.set[0].out) + row * a.set[0].ldo + f;
    T* const ok = static_cast<T*>(a.set[1].out) + row * a.set[1].ldo + (f - hq * a.d);
    for (int b = 0; run0 + b < run1; b += KI * step) {
      const bool more = run0 + b + KI * step < run1;  // heads of this token after the batch
#pragma unroll
      for (int k = 0; k < KI; ++k) {
        const int h = h0 + b + k * step;
        const bool second = h >= hq;
        float v[2 * E];
        V::unpack(raw[k][0], v);
        V::unpack(raw[k][1], v + E);
        if (more) load(xq, xk, h + KI * step, raw[k]);
        else if (next < tiles) load(nq, nk, h0 + k * step, raw[k]);
        if (run0 + b + k * step >= run1) continue;  // the same for the whole warp
        if constexpr (NORM != kNoNorm) {
          const float rd = 1.f / static_cast<float>(a.d);
          if constexpr (NORM == kLayer) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) sum += v[e];
            if (!active) sum = 0.f;
            for (int o = 1 << log_lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float mean = sum * rd;
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) v[e] -= mean;
          }
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 2 * E; ++e) ss = fmaf(v[e], v[e], ss);
          if (!active) ss = 0.f;
          for (int o = 1 << log_lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(fmaf(ss, rd, a.eps));
          const float4* w = wsm + (second ? 2 * Q * units : 0) + (active ? lane : 0);
#pragma unroll
          for (int j = 0; j < Q; ++j) {
            const float4 q = w[j * units];
            v[4 * j] *= inv * q.x, v[4 * j + 1] *= inv * q.y, v[4 * j + 2] *= inv * q.z, v[4 * j + 3] *= inv * q.w;
            if constexpr (NORM == kLayer) {
              const float4 r = w[(Q + j) * units];
              v[4 * j] += r.x, v[4 * j + 1] += r.y, v[4 * j + 2] += r.z, v[4 * j + 3] += r.w;
            }
          }
        }
        if (turned) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : E + e;
            const float x = v[ia], y = v[ib];
            v[ia] = x * c[e] - y * sn[e];
            v[ib] = y * c[e] + x * sn[e];
          }
        }
        if (mine && h < run1) {
          T* out = (second ? ok : oq) + h * a.d;
          *reinterpret_cast<Raw*>(out) = V::pack(v);
          *reinterpret_cast<Raw*>(out + gap) = V::pack(v + E);
        }
      }
    }
    xq = nq, xk = nk;
  }
}

template <typename T, int E, int NORM, bool INTER>
cudaError_t launch_vec(const RotaryArgs& a, cudaStream_t s) {
  constexpr int KI = 3;
  const int units = a.d / (2 * E), heads = a.set[0].heads + a.set[1].heads, half = a.rot / 2;
  int log_lanes = 0;
  while (1 << log_lanes < units) ++log_lanes;
  const int groups = 32 >> log_lanes, sms = num_sms_cached();
  // several tokens to a warp where one token's heads would leave groups or the KI
  // loads of a lane idle, as long as the SMs keep 8 warps each
  int log_tokens = 0;
  while (2 << log_tokens <= groups && (2ll << log_tokens) * heads <= static_cast<long long>(KI) * groups &&
         half << log_tokens <= 128 && a.T >> (log_tokens + 1) >= 8 * sms)
    ++log_tokens;
  // and a token's heads in several runs where the tokens are fewer than that
  const int batch = KI * (groups >> log_tokens);
  int runs = 1;
  while (runs < 64 && static_cast<long long>(a.T) * runs < 8 * sms && heads > batch * runs) ++runs;
  const int run = ((heads + runs - 1) / runs + batch - 1) / batch * batch;
  runs = (heads + run - 1) / run;
  const int tiles = (a.T - 1) / (1 << log_tokens) + 1;
  const size_t smem = (static_cast<size_t>(half) << log_tokens) * 64 + (NORM == kNoNorm ? 0 : 16 * a.d) + 8 * half;
  auto kern = rotary_vec_kernel<T, E, NORM, INTER, KI>;
  const dim3 grid(std::min((tiles - 1) / 8 + 1, sms * 4), runs);
  return launch_plain(kern, grid, dim3(256), smem, s, a, log_lanes, log_tokens, run);
}

// Whether heads, pairs and rows come apart into E-vectors, 32 units to a head at most.
bool vec_takes(const RotaryArgs& a, int E, int elem) {
  if (a.rot % (2 * E) || a.d % (2 * E) || a.d > 64 * E) return false;
  const long long heads = static_cast<long long>(a.set[0].heads) + a.set[1].heads;
  if (heads * a.d > INT_MAX) return false;  // 32-bit offsets inside a row, k's from hq heads before it
  for (const HeadSet& h : a.set) {
    if (h.heads == 0) continue;
    if ((reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.out)) % static_cast<unsigned>(E * elem))
      return false;
    if (a.T > 1 && (h.ldx % E || h.ldo % E)) return false;
    if (h.heads > 1 && (h.hsx % E || h.hsx * heads > INT_MAX)) return false;
  }
  return true;
}

template <typename T, int NORM>
cudaError_t launch_norm(const RotaryArgs& a, cudaStream_t s) {
  constexpr int kMost = 16 / static_cast<int>(sizeof(T));
  auto with = [&](auto e) {
    constexpr int E = decltype(e)::value;
    return a.interleaved ? launch_vec<T, E, NORM, true>(a, s) : launch_vec<T, E, NORM, false>(a, s);
  };
  if (vec_takes(a, kMost, sizeof(T))) return with(std::integral_constant<int, kMost>());
  if (vec_takes(a, kMost / 2, sizeof(T))) return with(std::integral_constant<int, kMost / 2>());
  if constexpr (sizeof(T) == 2)
    if (vec_takes(a, 2, sizeof(T))) return with(std::integral_constant<int, 2>());
  return launch_any<T, NORM>(a, s);
}

template <typename T>
cudaError_t launch_rotary(const RotaryArgs& a, int norm, cudaStream_t s) {
  switch (norm) {
    case kNoNorm: return launch_norm<T, kNoNorm>(a, s);
    case kRms: return launch_norm<T, kRms>(a, s);
    default: return launch_norm<T, kLayer>(a, s);
  }
}

int bad(const char* what, const char* why) {
  return record_error(INL_ERR_INVALID_INPUT, std::string(what) + ": " + why);
}

// Checks that need no device. Row widths as 64-bit products.
int check_rotary(const char* what, int dtype, int T, int d, int rot, const RotaryArgs& a) {
  if (dtype != INL_DTYPE_F32 && dtype != INL_DTYPE_BF16) return bad(what, "dtype is f32 or bf16");
  // a lane's feature index steps past d by up to 32
  if (T < 0 || T > 1 << 30 || d <= 0 || d > 1 << 30) return bad(what, "T from 0 to 2^30, d from 1 to 2^30");
  if (rot < 0 || rot > d || (rot & 1)) return bad(what, "rotary_dim is even and at most d");
  if (!std::isfinite(a.scale)) return bad(what, "scale is finite");
  for (const HeadSet& h : a.set) {
    if (h.heads < 0 || h.heads > 65536) return bad(what, "heads from 0 to 65536");
    if (h.heads == 0 || T == 0) continue;
    if (h.hsx < d) return bad(what, "the head stride is at least d");
    // 2^40 elements is above any device's memory and, with 2^16 heads, keeps the products in 64 bits
    if (h.hsx > (1ll << 40) || h.ldx > (1ll << 40) || h.ldo > (1ll << 40)) return bad(what, "strides below 2^40");
    if (T > 1 && (h.ldx < (h.heads - 1) * h.hsx + d || h.ldo < static_cast<long long>(h.heads) * d))
      return bad(what, "row strides are at least the row's width");
    if (!h.x || !h.out) return record_error(INL_ERR_CONFIG, std::string(what) + ": NULL input or output");
    if (h.x == h.out && ((T > 1 && h.ldx != h.ldo) || (h.heads > 1 && h.hsx != d)))
      return bad(what, "in place needs equal strides");
  }
  if (T > 0 && rot > 0 && (!a.pos || !a.inv_freq))
    return record_error(INL_ERR_CONFIG, std::string(what) + ": NULL pos or inv_freq");
  return INL_OK;
}

int run_rotary(const char* what, int dtype, int norm, RotaryArgs& a, cudaStream_t s) {
  int r = check_rotary(what, dtype, a.T, a.d, a.rot, a);
  if (r) return r;
  if (a.T == 0 || (a.set[0].heads == 0 && a.set[1].heads == 0)) return INL_OK;
  const int es = dtype == INL_DTYPE_BF16 ? 2 : 4;
  for (HeadSet& h : a.set)
    if (h.heads == 0) h.x = nullptr, h.out = nullptr, h.w = nullptr, h.b = nullptr;
  if (a.rot == 0) a.inv_freq = nullptr, a.pos = nullptr;
  const std::initializer_list<HookPtr> ptrs = {
      {a.set[0].x, es, "q"},   {a.set[1].x, es, "k"},   {a.set[0].out, es, "q_out"}, {a.set[1].out, es, "k_out"},
      {a.set[0].w, 4, "qw"},   {a.set[0].b, 4, "qb"},   {a.set[1].w, 4, "kw"},       {a.set[1].b, 4, "kb"},
      {a.pos, 4, "pos"},       {a.inv_freq, 8, "inv_freq"}};
  if ((r = check_aligned(what, ptrs)) || (r = check_reachable(what, ptrs))) return r;
  return launched(what, dtype == INL_DTYPE_BF16 ? launch_rotary<__nv_bfloat16>(a, norm, s)
                                                : launch_rotary<float>(a, norm, s));
}

double yarn_magnitude(double factor, double m) { return factor > 1.0 ? 0.1 * m * std::log(factor) + 1.0 : 1.0; }

int rope_frequencies(const inl_rope_config& c, double* inv_freq, float* scale) {
  const char* what = "rope_frequencies";
  const int rot = c.rotary_dim, half = rot / 2;
  if (rot <= 0 || (rot & 1) || rot > (1 << 20)) return bad(what, "rotary_dim is even and positive");
  if (!(c.theta > 0) || !std::isfinite(c.theta)) return bad(what, "theta is positive");
  for (double v : {c.factor, c.attention_factor, c.beta_fast, c.beta_slow, c.mscale, c.mscale_all_dim,
                   c.low_freq_factor, c.high_freq_factor})
    if (!std::isfinite(v) || v < 0) return bad(what, "factors are finite and not negative");
  const double factor = c.factor > 0 ? c.factor : 1.0;
  const double orig = c.original_max_position;
  constexpr double kTwoPi = 6.283185307179586476925287;
  if (c.type >= INL_ROPE_DYNAMIC && c.type <= INL_ROPE_LONGROPE && c.original_max_position < 1)
    return bad(what, "this type needs original_max_position");
  auto base = [&](double theta, int i) { return std::pow(theta, -2.0 * i / rot); };
  double mag = 1.0;
  std::vector<double> f(half);
  switch (c.type) {
    case INL_ROPE_DEFAULT:
      for (int i = 0; i < half; ++i) f[i] = base(c.theta, i);
      break;
    case INL_ROPE_LINEAR:
      for (int i = 0; i < half; ++i) f[i] = base(c.theta, i) / factor;
      break;
    case INL_ROPE_DYNAMIC: {
      if (rot < 4) return bad(what, "dynamic scaling needs rotary_dim >= 4");
      const double len = std::max<double>(c.seq_len, orig);
      const double grow = factor * len / orig - (factor - 1.0);
      if (!(grow > 0)) return bad(what, "dynamic scaling: factor below 1 for this length");
      const double theta = c.theta * std::pow(grow, rot / (rot - 2.0));
      for (int i = 0; i < half; ++i) f[i] = base(theta, i);
      break;
    }
    case INL_ROPE_YARN: {
      if (!(c.theta > 1)) return bad(what, "yarn needs theta > 1");
      const double fast = c.beta_fast > 0 ? c.beta_fast : 32.0, slow = c.beta_slow > 0 ? c.beta_slow : 1.0;
      auto pair_of = [&](double turns) {  // the (real) feature index / 2 that makes `turns` turns in `orig` positions
        return rot * std::log(orig / (turns * kTwoPi)) / (2.0 * std::log(c.theta));
      };
      double low = pair_of(fast), high = pair_of(slow);
      if (!c.no_truncate) low = std::floor(low), high = std::ceil(high);
      low = std::max(low, 0.0);
      high = std::min(high, rot - 1.0);
      if (low == high) high += 0.001;
      for (int i = 0; i < half; ++i) {
        const double ramp = std::min(std::max((i - low) / (high - low), 0.0), 1.0);
        const double b = base(c.theta, i);
        f[i] = b / factor * ramp + b * (1.0 - ramp);
      }
      mag = c.attention_factor > 0 ? c.attention_factor
            : c.mscale > 0 && c.mscale_all_dim > 0
                ? yarn_magnitude(factor, c.mscale) / yarn_magnitude(factor, c.mscale_all_dim)
                : yarn_magnitude(factor, 1.0);
      break;
    }
    case INL_ROPE_LLAMA3: {
      const double lo = c.low_freq_factor > 0 ? c.low_freq_factor : 1.0;
      const double hi = c.high_freq_factor > 0 ? c.high_freq_factor : 4.0;
      if (!(hi > lo)) return bad(what, "llama3 needs high_freq_factor > low_freq_factor");
      for (int i = 0; i < half; ++i) {
        const double b = base(c.theta, i);
        const double smooth = std::min(std::max((orig * b / kTwoPi - lo) / (hi - lo), 0.0), 1.0);
        f[i] = (1.0 - smooth) * b / factor + smooth * b;
      }
      break;
    }
    case INL_ROPE_LONGROPE: {
      const double* div = c.seq_len > c.original_max_position ? c.long_factor : c.short_factor;
      if (!div) return record_error(INL_ERR_CONFIG, "rope_frequencies: NULL short_factor or long_factor");
      for (int i = 0; i < half; ++i) {
        if (!(div[i] > 0) || !std::isfinite(div[i])) return bad(what, "longrope factors are positive");
        f[i] = base(c.theta, i) / div[i];
      }
      if (c.attention_factor > 0) {
        mag = c.attention_factor;
      } else if (factor > 1.0) {
        if (c.original_max_position < 2) return bad(what, "longrope needs original_max_position > 1");
        mag = std::sqrt(1.0 + std::log(factor) / std::log(orig));
      }
      break;
    }
    default: return bad(what, "unknown type");
  }
  for (int i = 0; i < half; ++i)
    if (!std::isfinite(f[i])) return bad(what, "theta and factors give a frequency that is not finite");
  std::copy(f.begin(), f.end(), inv_freq);
  *scale = static_cast<float>(mag);
  return INL_OK;
}

}  // namespace

}  // namespace inl

extern "C" {

int inl_cuda_rope_frequencies(const inl_rope_config* config, double* inv_freq, float* scale) {
  return inl::guarded([&] {
    if (!config || !inv_freq || !scale) return inl::record_error(INL_ERR_CONFIG, "rope_frequencies: NULL argument");
    return inl::rope_frequencies(*config, inv_freq, scale);
  });
}

int inl_cuda_rope(const void* x, int64_t ldx, int dtype, int T, int heads, int d, int rotary_dim, int interleaved,
                  const int32_t* pos, const double* inv_freq, float scale, int inverse, void* out, int64_t ldo,
                  void* stream) {
  return inl::guarded([&] {
    inl::RotaryArgs a{};
    a.set[0] = {x, out, nullptr, nullptr, ldx, d, ldo, heads};
    a.T = T, a.d = d, a.rot = rotary_dim, a.interleaved = interleaved != 0;
    a.scale = scale, a.sin_sign = inverse ? -1.f : 1.f;
    a.pos = pos, a.inv_freq = inv_freq;
    return inl::run_rotary("rope", dtype, inl::kNoNorm, a, static_cast<cudaStream_t>(stream));
  });
}

int inl_cuda_qk_norm_rotary(const void* q, int64_t ldq, int64_t q_head_stride, const void* k, int64_t ldk, int dtype,
                            int T, int hq, int hkv, int d, int layer_norm, const float* qw, const float* qb,
                            const float* kw, const float* kb, float eps, int rotary_dim, int interleaved,
                            const int32_t* pos, const double* inv_freq, float scale, void* q_out, int64_t ldqo,
                            void* k_out, int64_t ldko, void* stream) {
  return inl::guarded([&] {
    if (!layer_norm && (qb || kb)) return inl::bad("qk_norm_rotary", "a bias needs layer_norm");
    if (!(eps >= 0.f) || std::isinf(eps)) return inl::bad("qk_norm_rotary", "eps is finite and not negative");
    inl::RotaryArgs a{};
    a.set[0] = {q, q_out, qw, qb, ldq, q_head_stride, ldqo, hq};
    a.set[1] = {k, k_out, kw, kb, ldk, d, ldko, hkv};
    a.T = T, a.d = d, a.rot = rotary_dim, a.interleaved = interleaved != 0;
    a.eps = eps, a.scale = scale, a.sin_sign = 1.f;
    a.pos = pos, a.inv_freq = inv_freq;
    return inl::run_rotary("qk_norm_rotary", dtype, layer_norm ? inl::kLayer : inl::kRms, a,
                           static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
