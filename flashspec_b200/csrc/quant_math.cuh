// The affine INT8 format's arithmetic on the device, one element or 16 at a time.  Bit-exact
// with the reference (src/flashspec/quant.py:141-158): every operation is an explicitly
// rounded intrinsic, and files that include this must not be built with --use_fast_math.
#pragma once

#include <cuda_runtime.h>

#include <math.h>
#include <stdint.h>

namespace fsb {

struct QParams {
  float scale, zp;
};

__device__ __forceinline__ QParams qparams_from_range(float mn, float mx) {
  QParams q;
  q.scale = fmaxf(__fdiv_rn(__fsub_rn(mx, mn), 255.0f), 1.0e-8f);
  q.zp = fminf(fmaxf(rintf(__fdiv_rn(-mn, q.scale)), 0.0f), 255.0f);
  return q;
}

__device__ __forceinline__ int8_t quantize_one(float x, QParams q) {
  const float u = fminf(fmaxf(rintf(__fadd_rn(__fdiv_rn(x, q.scale), q.zp)), 0.0f), 255.0f);
  return (int8_t)((int)u - 128);
}

__device__ __forceinline__ float dequant_one(int8_t v, float scale, int16_t zp) {
  return __fmul_rn(__fsub_rn((float)((int)v + 128), (float)zp), scale);
}

// Out of line so that the unrolled fast path carries one copy of the division.
static __device__ __noinline__ int8_t quantize_one_exact(float x, QParams q) { return quantize_one(x, q); }

// 16 x quantize_one, bit-identical, packed as 16 int8 bytes, with almost no divisions.
//   qa = RN(x * RN(1/s)) is within |x/s| (2^-23 + 2^-24 + 2^-47) of q = RN(x/s) (1/s is a
//   normal float: 1e-8 <= s < 2^128 / 255), so wherever ta = RN(qa + zp) lies in [0, 255]
//   (|q| < 511) it is within 1.0e-4 + ulp(ta) < 1.4e-4 of t = RN(q + zp).  The reference
//   code is clamp(rint(t), 0, 255) = rint(clamp(t, 0, 255)) (integer bounds); rint is
//   constant between half-integers, so when tc = clamp(ta, 0, 255) lies more than 2^-11
//   (4.9e-4) from the nearest half-integer the code is rint(tc), and a ta that clamps is
//   off by less than the margin from a t that clamps the same way.  rint(tc) is the low
//   byte of RN(tc + 1.5 * 2^23) (round-to-nearest-even, tc < 2^22), d = tc - rint(tc) is
//   exact, and the elements with |d| >= 0.5 - 2^-11 (about 0.1%) take the division.
//   NaN: fmaxf(NaN, 0) = 0, the same code as the division path gives.
__device__ __forceinline__ uint4 quantize16_fast(const float* v, QParams q) {
  const float rcp = __frcp_rn(q.scale);
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  uint32_t bits[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float ta = __fadd_rn(__fmul_rn(v[j], rcp), q.zp);
    const float tc = fminf(fmaxf(ta, 0.0f), 255.0f);
    const float r = __fadd_rn(tc, kMagic);
    const float d = __fsub_rn(tc, __fsub_rn(r, kMagic));
    bits[j] = __float_as_uint(r);  // low byte = rint(tc)
    if (fabsf(d) >= 0.5f - 4.8828125e-4f) bits[j] = (uint32_t)(uint8_t)quantize_one_exact(v[j], q) ^ 0x80u;
  }
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = __byte_perm(bits[4 * k], bits[4 * k + 1], 0x0040);
    const uint32_t hi = __byte_perm(bits[4 * k + 2], bits[4 * k + 3], 0x0040);
    w[k] = __byte_perm(lo, hi, 0x5410) ^ 0x80808080u;  // code - 128 as int8
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// dequant_one of the 16 int8 codes in raw, bit-identical: the byte u = code + 128 is put
// in the mantissa of 2^23 (the float 2^23 + u, exact), and (2^23 + u) - (2^23 + zp) = u - zp
// exactly (|zp| < 2^23), which is dequant_one's first step; then the same RN product.
__device__ __forceinline__ void dequant16(int4 raw, float scale, int16_t zp, float* out) {
  const float base = __fadd_rn(8388608.0f, (float)zp);
  const uint32_t w4[4] = {(uint32_t)raw.x ^ 0x80808080u, (uint32_t)raw.y ^ 0x80808080u,
                          (uint32_t)raw.z ^ 0x80808080u, (uint32_t)raw.w ^ 0x80808080u};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float f = __uint_as_float(__byte_perm(w4[j >> 2], 0x4B000000u, 0x7540 | (j & 3)));
    out[j] = __fmul_rn(__fsub_rn(f, base), scale);
  }
}

}  // namespace fsb
