// The 8-bit form of a cached row (one token's key or value of one head): a 32-bit scale and a signed 8-bit code per number,
//     scale = max(amax / 127, 2^-120),   code = the whole number nearest to x / scale, ties to even,   value = code * scale.
// The code is the one nearest by the exact quotient, not by a rounded one: half steps are common (x = amax / 2 is one, and 16-bit
// rows hold it often), and there a rounded quotient gives one code or the other by chance.  A row with an infinity or a NaN has
// scale NaN and codes 0: every value read back from it is NaN.  The floor of the scale keeps its reciprocal finite; numbers below
// 2^-121 are read back as 0.
#pragma once
#include "common.cuh"
#include "packed.cuh"

namespace cbis {

// A number of a call's record as an int: what lies beyond 2^30 (behind every position) is 2^30 + 1, below -2^30 it is -2^30 - 1.
inline int q8_int(long long x) {
  const long long most = (1 << 30) + 1;
  return (int)(x > most ? most : (x < -most ? -most : x));
}

constexpr float Q8_FLOOR = 7.52316384526264e-37f;      // 2^-120

// The largest magnitude as the bits of |x|: ordered like the magnitudes, an infinity above every number and a NaN above that.
__device__ __forceinline__ unsigned q8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// amax / 127 rounded to nearest: the product with 1 / 127 and what it leaves over, times 1 / 127 again (Markstein's correction of a
// quotient: with a correctly rounded reciprocal the second sum is the correctly rounded quotient).
__device__ __forceinline__ float q8_scale(unsigned amax_bits) {
  const float a = __uint_as_float(amax_bits), c = 1.f / 127.f, q = a * c;
  return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(fmaf(fmaf(-q, 127.f, a), c, q), Q8_FLOOR);
}
// 1 / scale to 2^-22 or so: the exact way below needs no more.
__device__ __forceinline__ float q8_inverse(float scale) { return __frcp_rn(scale); }

// The codes of four numbers, a byte each.  Adding 1.5 * 2^23 rounds x / scale to a whole number, ties to even, and leaves it in the low
// bits; the quotient is a product with the reciprocal, good to 2^-22, so only a number that close to a half step needs the exact way.
__device__ __forceinline__ int q8_code(float x, float scale, float inv);
__device__ __forceinline__ unsigned q8_codes4(const float* x, float scale, float inv) {
  float f[4], far = 0.f;
  const unsigned long long inv2 = pack2(inv, inv), up = pack2(12582912.f, 12582912.f), down = pack2(-12582912.f, -12582912.f), neg = pack2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const unsigned long long y = mul2(pack2(x[i], x[i + 1]), inv2), z = add2(y, up);
    float d0, d1;
    unpack2(z, f[i], f[i + 1]);
    unpack2(fma2(add2(z, down), neg, y), d0, d1);
    far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
  }
  if (far > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)q8_code(x[i], scale, inv) + 12582912.f;
  }
  const unsigned w = __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040),
                                 __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040), 0x5410);
  return scale == scale ? w : 0u;
}

// The same one by one.  inv: the reciprocal of the scale.  q is at most one step off; the remainder x - q scale is exact in 32 bits.
__device__ __forceinline__ int q8_code(float x, float scale, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, scale, x), half = 0.5f * scale;
  const bool odd = ((int)q & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.f;
  if (r < -half || (r == -half && odd)) q -= 1.f;
  return scale == scale ? (int)q : 0;
}

}  // namespace cbis
