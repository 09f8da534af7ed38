// Activations held in whole numbers of 8 or 16 bits, of which 32 along the last dim share a power of two (8 bits: MXINT8 of the OCP Microscaling Formats
// specification, version 1.0).  With n = 6 or 14:
//
//   e = max(floor(log2 of the largest magnitude), n - 126)     code = v 2^(n-e), rounded to even, within +-(2^(n+1) - 1)     value = code 2^(e-n)
//
// The scale byte is e + 127; a block with an infinity or a NaN has the byte 255 and reads as NaN.  The format's e goes down to -127; what is written here stops where
// the unit is 2^-126, so every value is a normal fp32 number, and with 8 bits exact in bf16: products of the values on the tensor cores lose nothing to the format.
// What is read may come from elsewhere and have any byte; 8-bit values below 2^-126 are multiples of 2^-133, exact in both types too.
//
// MX_HALF: fp16 numbers under the block's power of two, v 2^(14-e), with n = 14 otherwise.  A value keeps its own exponent: it is off by at most 2^-11 of itself
// down to 2^-28 of its block's largest (bf16: 2^-8), and by 2^-39 of that below; whole numbers of 16 bits are off by 2^-15 of the block's largest, whatever the value.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace apb {

constexpr int MX_BLOCK = 32, MX_NAN = 255;
constexpr int MX_HALF = 11;  // (as BITS: those of a value)
template <int BITS>
constexpr int MX_BYTES = BITS == 8 ? 1 : 2;  // of a code
template <int BITS>
constexpr int MX_LOWEST = 8 * MX_BYTES<BITS> - 1;  // the scale byte of the smallest e

// What the values of a block are multiplied with to be codes, 2^(n - e), or 0 where it holds an infinity or a NaN.  (bytes from MX_LOWEST on: a normal number)
template <int BITS>
__device__ __forceinline__ float mx_to_code(uint32_t byte) {
  return __uint_as_float(byte == MX_NAN ? 0u : (uint32_t)(252 + 8 * MX_BYTES<BITS> - (int)byte) << 23);
}
// 2^e, or NaN, of any byte: the format's own conversion, exact in bf16.  (For byte 0 below the normal numbers; in files compiled with fast math that is zero.)
__device__ __forceinline__ float mx_power(uint32_t byte) { return __uint_as_float((uint32_t)__nv_cvt_e8m0_to_bf16raw((__nv_fp8_storage_t)byte).x << 16); }
__device__ __forceinline__ float mx_bits(uint32_t v) { return __uint_as_float(v); }

// ``top``: the largest of the magnitudes' bits, in which a NaN is larger than everything.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t field = top >> 23;
  return field == 255 ? MX_NAN : field < MX_LOWEST<BITS> ? MX_LOWEST<BITS> : field;
}

// Largest magnitude (its bits) of 32 values, of which a NaN is larger than everything; four chains, as one would wait for itself.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t mx_top(const uint32_t (&r)[32]) {
  float top[4] = {};
#pragma unroll
  for (int i = 0; i < 32; ++i) top[i & 3] = max_nan(top[i & 3], fabsf(__uint_as_float(r[i])));
  return __float_as_uint(max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])));
}

// Values of one block to codes.  Added to 1.5 2^23, a number below 2^22 is rounded to a whole one, ties to even, whose lower bits are the code: one addition
// with the scaling, and a byte permutation for two codes.  What rounds to 2^(n+1) is clamped, and a broken block has codes of zero: ``exact`` says that
// neither occurs, which is so where the block's largest value does not round so high.
template <int BITS>
struct MxCoder {
  static constexpr float ROUND = 12582912.f, LIMIT = (1 << (BITS - 1)) - 1;
  static constexpr uint32_t TIE = BITS == 8 ? 0x7f0000u : 0x7fff00u;  // the mantissa of 2^(n+1) - 1/2
  float m;
  bool exact;
  __device__ __forceinline__ MxCoder(uint32_t byte, uint32_t top)
      : m(mx_to_code<BITS>(byte)), exact(byte != MX_NAN && (top & 0x7fffffu) < TIE) {}
  template <bool EXACT>
  __device__ __forceinline__ float add(uint32_t bits) const {
    const float f = mx_bits(bits);
    return EXACT ? fmaf(f, m, ROUND) : ROUND + (m == 0.f ? 0.f : fminf(LIMIT, fmaxf(-LIMIT, f * m)));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {  // four lowest bytes
    const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410); }  // two lower halves
  // four codes of 8 bits, two of 16
  template <bool EXACT>
  __device__ __forceinline__ uint32_t word(const uint32_t* v) const {
    if constexpr (BITS == 8) return pack(add<EXACT>(v[0]), add<EXACT>(v[1]), add<EXACT>(v[2]), add<EXACT>(v[3]));
    else return pack(add<EXACT>(v[0]), add<EXACT>(v[1]));
  }
  // ``n`` words of codes; one branch for all of them
  template <int n>
  __device__ __forceinline__ void words(const uint32_t* v, uint32_t (&w)[n]) const {
    if (exact) {
#pragma unroll
      for (int i = 0; i < n; ++i) w[i] = word<true>(v + 32 / BITS * i);
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) w[i] = word<false>(v + 32 / BITS * i);
    }
  }
};
template <>
struct MxCoder<MX_HALF> {
  float m;
  __device__ __forceinline__ MxCoder(uint32_t byte, uint32_t) : m(mx_to_code<MX_HALF>(byte)) {}
  template <int n>
  __device__ __forceinline__ void words(const uint32_t* v, uint32_t (&w)[n]) const {
    if (m != 0.f) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const __half2 h = __floats2half2_rn(mx_bits(v[2 * i]) * m, mx_bits(v[2 * i + 1]) * m);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    } else {  // (a broken block)
#pragma unroll
      for (int i = 0; i < n; ++i) w[i] = 0;
    }
  }
};

// Codes of one block to values: with 2^(n+1) added, a code is the lowest byte (or two) of 2^23 + (code + 2^(n+1)) as fp32; one permutation, an FMA for code 2^-n and a
// multiplication by 2^e, both exact.  (In one step, with 2^23 + 2^(n+1) times the power of two taken off, that product would be infinite from e = 111 on, or 119.
// 2^(e-n) instead of 2^e, with the comparison that bytes below n need: 8192 x 14343 back 101 -> 113 us.)
template <int BITS>
struct MxReader {
  static constexpr float UNIT = BITS == 8 ? 0x1p-6f : 0x1p-14f, BIAS = (8388608.f + (1 << (BITS - 1))) * UNIT;
  float m;
  MxReader() = default;
  __device__ __forceinline__ explicit MxReader(uint32_t byte) : m(mx_power(byte)) {}
  __device__ __forceinline__ void four(uint32_t codes, float* f) const {  // (8 bits)
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fmaf(mx_bits(__byte_perm(u, 0x4b000000u, 0x7440 | i)), UNIT, -BIAS) * m;
  }
  __device__ __forceinline__ void two(uint32_t codes, float* f) const {  // (16 bits)
    const uint32_t u = codes ^ 0x80008000u;
    f[0] = fmaf(mx_bits(__byte_perm(u, 0x4b000000u, 0x7410)), UNIT, -BIAS) * m;
    f[1] = fmaf(mx_bits(__byte_perm(u, 0x4b000000u, 0x7432)), UNIT, -BIAS) * m;
  }
};
template <>
struct MxReader<MX_HALF> {
  float m;
  MxReader() = default;
  __device__ __forceinline__ explicit MxReader(uint32_t byte) : m(mx_power(byte) * 0x1p-14f) {}
  __device__ __forceinline__ void two(uint32_t codes, float* f) const {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&codes));
    f[0] = v.x * m;
    f[1] = v.y * m;
  }
};

}  // namespace apb
