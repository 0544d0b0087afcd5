// The block formats of the 8-bit operators: 8-bit floating-point values (OCP e4m3 and e5m2) and one power of two for each block
// of them, held as its biased exponent in a byte: value = code * 2^(byte - 127).
//
// The byte of a block is the smallest, from 1 on, with which its largest magnitude is at most 1.75 * 2^TOP, the largest value
// of the format (e4m3 448: TOP 8; e5m2 57344: TOP 15), so nothing saturates.  A power of two because scaling by it is exact,
// on the way in, in the matrix instructions (which take such bytes as operands) and on the way out; a scale with a mantissa
// would place the largest value at the format's end, a gain of at most one step in the range, none in the precision.
#pragma once
#include "pk_common.h"

namespace pk_fp8 {

constexpr int TOP_E4M3 = 8, TOP_E5M2 = 15;
constexpr uint32_t INF_BITS = 0x7f800000u, NAN_CODE = 0x7fu;

// bits: a finite magnitude's
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits, int top) {
  const int s = (int)(bits >> 23) - top + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(s < 1 ? 1 : s);
}
// 2^(byte - 127) and 2^(127 - byte), byte 1 to 253 (a byte of 0 stands for 0)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float inverse_scale_of(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// The largest of 16 neighbouring lanes' values (a row of the data-parallel primitives), in every one of them: rotations by 8
// and 4, then within quads.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#define PK_STEP(CTRL)                                                                                \
  {                                                                                                  \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); \
    v = o > v ? o : v;                                                                               \
  }
  PK_STEP(0x128) PK_STEP(0x124) PK_STEP(0x4e) PK_STEP(0xb1)
#undef PK_STEP
  return v;
}
// Four e4m3 codes of values of at most 448, rounded to nearest even (half a step, 2^-4 of the value: the products of a block
// average such errors, and nothing here is summed up over steps).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// What a block of largest magnitude `bits` is divided by.  A block with an infinity or a NaN is NaN throughout, so that its rows'
// products are.
struct BlockScale {
  uint32_t byte;
  float inverse;
  bool finite;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t bits) {
  BlockScale s;
  s.finite = bits < INF_BITS;
  s.byte = s.finite ? scale_byte(bits, TOP_E4M3) : 127u;
  s.inverse = inverse_scale_of(s.byte);
  return s;
}
// 16 values of a block
__device__ __forceinline__ u32x4_t codes16(const float (&f)[16], const BlockScale& s) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = s.finite ? e4m3x4(f[4 * i] * s.inverse, f[4 * i + 1] * s.inverse, f[4 * i + 2] * s.inverse, f[4 * i + 3] * s.inverse)
                    : NAN_CODE * 0x01010101u;
  return v;
}

// Eight neighbouring values of a lane and those of the 15 lanes beside it are one block of 128: its codes and its byte.
__device__ __forceinline__ void quantize8(const float (&f)[8], uint32_t (&codes)[2], uint32_t& byte) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  const BlockScale s = block_scale(row_max(m));
  byte = s.byte;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    codes[i] = s.finite ? e4m3x4(f[4 * i] * s.inverse, f[4 * i + 1] * s.inverse, f[4 * i + 2] * s.inverse, f[4 * i + 3] * s.inverse)
                        : NAN_CODE * 0x01010101u;
}

}  // namespace pk_fp8
