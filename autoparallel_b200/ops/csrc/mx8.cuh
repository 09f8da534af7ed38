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

// Largest magnitude (its bits) of 32 values, of which a NaN is larger than everything.
__device__ __forceinline__ uint32_t mx8_top(const uint32_t (&r)[32]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(__uint_as_float(r[i]))));
  return __float_as_uint(top);
}

// Values of one block to codes.  Added to 1.5 2^23, a number below 2^22 is rounded to a whole one, ties to even, whose lower byte is the code; one addition
// with the scaling, one byte permutation for two codes.  What rounds to 128 is clamped, and a broken block has codes of zero: ``exact`` says that neither
// occurs, which is so where the block's largest value does not round to 128.
struct Mx8Coder {
  float m;
  bool exact;
  __device__ __forceinline__ Mx8Coder(uint32_t byte, uint32_t top) : m(mx8_to_code(byte)), exact(byte != MX8_NAN && (top & 0x7fffffu) < 0x7f0000u) {}
  static constexpr float ROUND = 12582912.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {  // lowest bytes
    const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  __device__ __forceinline__ uint32_t four(uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
    float f[4] = {__uint_as_float(a), __uint_as_float(b), __uint_as_float(c), __uint_as_float(d)};
    if (!exact) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = m == 0.f ? 0.f : fminf(127.f, fmaxf(-127.f, f[i] * m));
    }
    const float k = exact ? m : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fmaf(f[i], k, ROUND);
    return pack(f[0], f[1], f[2], f[3]);
  }
};

// Codes of one block to values: with 128 added, a code is the lowest byte of 2^23 + (code + 128) as fp32; one permutation, and a multiplication by the power
// of two that takes 2^23 + 128 times it off again, exactly.
struct Mx8Reader {
  float m, off;
  Mx8Reader() = default;
  __device__ __forceinline__ explicit Mx8Reader(uint32_t byte) : m(mx8_to_value(byte)), off(-8388736.f * m) {}
  __device__ __forceinline__ void four(uint32_t codes, float* f) const {
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fmaf(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | i)), m, off);
  }
};

}  // namespace apb
