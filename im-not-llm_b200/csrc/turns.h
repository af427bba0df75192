// Angles of rotary positions, to 32-bit cosines and sines: on the device, and on
// the host for tests.
#pragma once

#include <math.h>
#include <stdint.h>

#ifdef __CUDACC__
#define INL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define INL_HOST_DEVICE inline
#endif

namespace inl {

// inv_freq (radians per position) as a fraction of a turn per position in
// 2^-64 turns: pos times it, modulo 2^64, is where the angle ends in its turn,
// exactly, for any 32-bit position, by one integer product.
INL_HOST_DEVICE uint64_t turn_step(double inv_freq) {
  const double turns = inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  const double part = turns - floor(turns);  // a whole turn just below zero; NaN where inv_freq is not finite
  return part < 1.0 ? static_cast<uint64_t>(part * 18446744073709551616.0) : 0;
}

// cos and sin of the angle pos * step: the quarter turn nearest to it by
// integer arithmetic, and the rest, at most an eighth of a turn, by the Taylor
// polynomials (the first terms left out are below 2e-9).
INL_HOST_DEVICE void turn_of(int pos, uint64_t step, float& c, float& s) {
  const int t = static_cast<int>((static_cast<uint64_t>(static_cast<long long>(pos)) * step) >> 32);
  // wraps to the same quarter at half a turn
  const int k = static_cast<int>(static_cast<unsigned>(t) + (1u << 29)) >> 30;
  const float x = static_cast<float>(static_cast<int>(static_cast<unsigned>(t) - (static_cast<unsigned>(k) << 30))) *
                  1.4629180792671596e-9f;  // 2 pi / 2^32
  const float x2 = x * x;
  float cr = fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f);
  cr = fmaf(x2, cr, -1.f / 720.f);
  cr = fmaf(x2, cr, 1.f / 24.f);
  cr = fmaf(x2, cr, -0.5f);
  cr = fmaf(x2, cr, 1.f);
  float sr = fmaf(x2, 1.f / 362880.f, -1.f / 5040.f);
  sr = fmaf(x2, sr, 1.f / 120.f);
  sr = fmaf(x2, sr, -1.f / 6.f);
  sr = fmaf(x2 * x, sr, x);
  const float p = (k & 1) ? sr : cr, q = (k & 1) ? cr : sr;
  c = ((k + 1) & 2) ? -p : p;
  s = (k & 2) ? -q : q;
}

}  // namespace inl
