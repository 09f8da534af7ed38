// Activations held in 8 bits (MXINT8 of the OCP Microscaling Formats specification, version 1.0): 32 values along the last dim share a power of two.
//
//   e = max(floor(log2 of the largest magnitude), -120)     code = v 2^(6-e), rounded to even, within +-127     value = code 2^(e-6)
//
// The scale byte is e + 127; a block with an infinity or a NaN has the byte 255 and reads as NaN.  A code has at most seven bits and e - 6 >= -126, so
// every value is exact in bf16, and products of the values on the tensor cores lose nothing to the format.
#pragma once
#include <stdint.h>

namespace apb {

constexpr int MX8_BLOCK = 32, MX8_NAN = 255, MX8_LOWEST = 7;  // (the last: the scale byte of e = -120)

// ``top``: the largest of the magnitudes' bits, in which a NaN is larger than everything.
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t top) {
  const uint32_t field = top >> 23;
  return field == 255 ? MX8_NAN : field < MX8_LOWEST ? MX8_LOWEST : field;
}
// 2^(6-e) and 2^(e-6)
__device__ __forceinline__ float mx8_to_code(uint32_t byte) { return byte == MX8_NAN ? 0.f : __uint_as_float((260u - byte) << 23); }
__device__ __forceinline__ float mx8_to_value(uint32_t byte) { return __uint_as_float(byte == MX8_NAN ? 0x7fc00000u : (byte - 6u) << 23); }

// A broken block has codes of zero: zero times an infinity would be a NaN, which converts to zero as well.
__device__ __forceinline__ uint32_t mx8_code(float v, float to_code) {
  const int c = __float2int_rn(v * to_code);
  return (uint32_t)max(-127, min(127, c)) & 255u;
}
__device__ __forceinline__ uint32_t mx8_codes4(float a, float b, float c, float d, float to_code) {
  return mx8_code(a, to_code) | mx8_code(b, to_code) << 8 | mx8_code(c, to_code) << 16 | mx8_code(d, to_code) << 24;
}
__device__ __forceinline__ float mx8_value(uint32_t word, int i, float to_value) { return (float)(int)(int8_t)(word >> (8 * i)) * to_value; }

}  // namespace apb
