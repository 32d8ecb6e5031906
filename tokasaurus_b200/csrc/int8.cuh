// Numbers held in 8 bits: a code in [-127, 127] times a float32 scale, scale = max|x| * (1 / 127), code = rint(x / scale).
#pragma once
#include "common.cuh"

namespace tkb {

constexpr float ONE_127TH = 1.f / 127.f;

// rint(x / s) with the quotient rounded as float32 division rounds it, held to [-127, 127].  A call: a division in place for every
// number of an unrolled loop is what such a kernel then waits for, as instructions.
__device__ __noinline__ int divided_code(float x, float s) { return (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f); }

// The same without a division, for 2^-100 <= s, as the bits of code + 1.5 * 2^23.  h, the half integer next to the quotient, parts the two
// codes that it may have; |x| - |h| s is exact where the quotient is close to h (a multiple of half a unit of s, few of them), and the
// rounded quotient is h itself within half a unit of h, which goes to the even code.
__device__ __forceinline__ uint32_t settled_code(float x, float s, float inv) {
  constexpr float ROUND = 12582912.f;
  const float t = x * inv, r = (t + ROUND) - ROUND, h = fabsf(r + copysignf(0.5f, t - r));
  const float off = fmaf(-h, s, fabsf(x)), above = __uint_as_float(__float_as_uint(h) & 0x7f800000u) * (s * 0x1p-24f);
  const float below = h == 0.5f ? 0.5f * above : above;  // (units halve below a power of two; the other powers are no half integers)
  return __float_as_uint(copysignf(h + (off > above ? 0.25f : off < -below ? -0.25f : 0.f), x) + ROUND);
}

// The codes of four numbers under scale s (> 0) as the bytes of a word; inv: 1 / s.  x * inv is within 3e-5 of the quotient, which
// settles all but those next to a half (2 in 10,000; of bfloat16 numbers, whose quotients are often such, 25) and those of a scale whose
// reciprocal is infinite.  Adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits (rintf and
// a conversion to int take the unit that has a quarter of the rate).
__device__ __forceinline__ uint32_t four_codes(const float4 x, float s, float inv) {
  constexpr float ROUND = 12582912.f;
  const float v[4] = {x.x, x.y, x.z, x.w};
  uint32_t b[4];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float t = v[i] * inv, r = t + ROUND;
    b[i] = __float_as_uint(r);
    near |= !(fabsf(t - (r - ROUND)) <= 0.4999f);  // (or no number, of an infinite reciprocal)
  }
  if (near) {
    if (s >= 0x1p-100f) {
#pragma unroll
      for (int i = 0; i < 4; i++) b[i] = settled_code(v[i], s, inv);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) b[i] = (uint32_t)divided_code(v[i], s);
    }
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
// Magnitudes as integers: NaN > infinity > every number.
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr unsigned NOT_FINITE = 0x7f800000u;  // magnitudes from here on

}  // namespace tkb
