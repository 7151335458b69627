// Rows of 8-bit integers with a 32-bit scale each: row r stands for q[r, k] * scale[r].
//
//   A = max(max_k |x_k|, 127 * 2^-126),   scale = A / 127,   q_k = 127 x_k / A rounded to nearest even
//
// The quotient is rounded as if it were exact, so a row's integers are a function of its values alone,
// whichever kernel made them.  (16-bit data has many quotients that end in one half: x = max / 2 gives 63.5.)
// The floor under A keeps scale a normal number and 127 / A finite; a row of zeros gets zeros.
// A row that holds a NaN or an infinity has no scale: it gets NaN, and zeros for q, so that whatever is
// computed from the row is NaN instead of wrong.
#pragma once
#include "common.cuh"

namespace skyla {
namespace q8 {

constexpr float kMost = 127.f;
constexpr float kLeastMax = 127.f * 1.17549435e-38f;  // 127 * 2^-126: exact
constexpr unsigned kInfBits = 0x7f800000u;
constexpr float kNan = __builtin_nanf("");

// |v| as bits: ordered like the values, an infinity above every number and a NaN above that
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Step {
  float most;  // A
  float inv;   // 127 / A, rounded
};
__device__ __forceinline__ Step step_of(unsigned max_bits) {
  Step s;
  s.most = fmaxf(__uint_as_float(max_bits), kLeastMax);
  s.inv = kMost / s.most;
  return s;
}

// 127 x / A is nearer to one half than 32 bits can tell: 254 |x| against (2 k + 1) A decides, both exact in
// 64 bits (k = the whole part).
__device__ __noinline__ int round_close(float x, float most, float z) {
  const int k = (int)fabsf(z);
  const double two_x = 254.0 * (double)fabsf(x), edge = (double)(2 * k + 1) * (double)most;
  const int n = two_x > edge ? k + 1 : (two_x < edge ? k : k + (k & 1));
  return x < 0.f ? -n : n;
}
// x * inv is within z * 2^-24 of the exact quotient z (inv's rounding), so its nearest integer is z's unless z lies
// that near to a half; 2^-15 is asked for.  Adding 1.5 * 2^23 rounds to an integer (to even) and leaves it in the low
// bits; d is what it moved by.
// HALVES: the values are bfloat16.  Then x = b 2^f and A = a 2^e with whole a, b < 256, and z is a half or at least
// z / (254 b) > z * 2^-16 from one, which the error cannot bridge: what lies within n * 2^-20 of a half is one, and
// goes to the even neighbour, twice the nearest integer of z / 2.  (They are common: x = A / 2 is one, and where
// a = 127 every second step.  Among 2,048 x 12,288 normal values the 64-bit comparison took every second warp's time:
// 23.3 us.)
template <int E, bool HALVES>
__device__ __forceinline__ void round_q(const float* x, const Step& s, uint32_t* n) {
  constexpr float kMagic = 12582912.f, kNear = 0.5f - 0x1p-15f;
  bool close = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float m = fmaf(x[i], s.inv, kMagic), d = fmaf(x[i], s.inv, kMagic - m);
    n[i] = __float_as_uint(m);
    close |= fabsf(d) > kNear;
  }
  if (close) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float m = fmaf(x[i], s.inv, kMagic), d = fmaf(x[i], s.inv, kMagic - m);
      if (HALVES) {
        if (fabsf(d) > fmaf(fabsf(kMagic - m), -0x1p-20f, 0.5f)) n[i] = __float_as_uint(fmaf(x[i], 0.5f * s.inv, kMagic)) << 1;
      } else {
        if (fabsf(d) > kNear) n[i] = (uint32_t)round_close(x[i], s.most, x[i] * s.inv);
      }
    }
  }
}
// the low bytes of four words
__device__ __forceinline__ uint32_t low_bytes(const uint32_t* n) {
  return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
}

// A product's sum with its two scales, in one order and never contracted into an addition that follows: every
// kernel of the 8-bit product gives the same bits.
__device__ __forceinline__ float scaled(int acc, float x_scale, float w_scale) {
  return __fmul_rn(__fmul_rn(__int2float_rn(acc), x_scale), w_scale);
}
// silu(g) u of a gated product, also one for all kernels.  With the fast exponential and division: their error (a few
// 2^-22; the exponential's grows with its argument, to 2^-16 at -87) is well below the bfloat16 rounding that follows.
// Gates below -87.3, where 1 + exp(-g) passes 2^126 and silu is below 2^-119, give zero.
__device__ __forceinline__ float silu_times(float g, float u) { return __fmul_rn(__fdividef(g, 1.0f + __expf(-g)), u); }

}  // namespace q8
}  // namespace skyla
