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
#include <cmath>
#include <string>
#include <vector>

#include "../../include/inl_cuda.h"
#include "../../include/inl_cuda_kernels.h"
#include "common.cuh"
#include "hook_checks.h"
#include "kernels.h"

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

// cos and sin of pos * inv_freq.
__device__ __forceinline__ void turn_of(int pos, double inv_freq, float& c, float& s) {
  const double quarter = static_cast<double>(pos) * inv_freq * 0.63661977236758134308;  // 2 / pi
  const double q = rint(quarter);
  const float r = static_cast<float>(quarter - q) * 0.5f;  // half turns, |r| <= 1/4
  float cr, sr;
  sincospif(r, &sr, &cr);
  const int k = static_cast<int>(static_cast<long long>(q)) & 3;
  const float a = (k & 1) ? sr : cr, b = (k & 1) ? cr : sr;
  c = (k == 1 || k == 2) ? -a : a;
  s = (k & 2) ? -b : b;
}

// Any head width, stride and alignment: a warp per (token, head), a lane per
// pair (and per feature that is copied), so that in-place rows are read and
// written by one lane alone. Two passes over the head when it is normed.
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
    const int pos = a.pos[t];
    for (int i = lane; i < half; i += 32) {
      const int ja = a.interleaved ? 2 * i : i, jb = a.interleaved ? 2 * i + 1 : i + half;
      float c, s;
      turn_of(pos, a.inv_freq[i], c, s);
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
  rotary_any_kernel<T, NORM><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rotary(const RotaryArgs& a, int norm, cudaStream_t s) {
  switch (norm) {
    case kNoNorm: return launch_any<T, kNoNorm>(a, s);
    case kRms: return launch_any<T, kRms>(a, s);
    default: return launch_any<T, kLayer>(a, s);
  }
}

int bad(const char* what, const char* why) {
  return record_error(INL_ERR_INVALID_INPUT, std::string(what) + ": " + why);
}

// Checks that need no device. Row widths as 64-bit products.
int check_rotary(const char* what, int dtype, int T, int d, int rot, const RotaryArgs& a) {
  if (dtype != INL_DTYPE_F32 && dtype != INL_DTYPE_BF16) return bad(what, "dtype is f32 or bf16");
  if (T < 0 || d <= 0) return bad(what, "T >= 0 and d > 0");
  if (rot < 0 || rot > d || (rot & 1)) return bad(what, "rotary_dim is even and at most d");
  if (!std::isfinite(a.scale)) return bad(what, "scale is finite");
  for (const HeadSet& h : a.set) {
    if (h.heads < 0) return bad(what, "heads >= 0");
    if (h.heads == 0 || T == 0) continue;
    if (h.hsx < d) return bad(what, "the head stride is at least d");
    // 2^40 elements is above any device's memory and keeps the products in 64 bits
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
  if (a.rot == 0) a.inv_freq = nullptr;
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
