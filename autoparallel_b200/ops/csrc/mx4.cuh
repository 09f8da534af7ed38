// What the kernels of microscaled 4-bit floating point share: the conversions, the layout in memory and in a stage of the products (see ops/mx4_ops.py).
#pragma once
#include <type_traits>

#include "gemm_core.cuh"

namespace apb {

// 8 values to 4 bytes of codes: value 2i in the low half of byte i
__device__ __forceinline__ uint32_t mx_encode(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// The code s e e m of a value v, moved to the top of an fp32 mantissa and the bottom of its exponent, is v * 2^-126, exactly (0.5 as a denormal).
__device__ __forceinline__ void mx_decode(uint32_t codes, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = codes >> (4 * i);
    v[i] = (__uint_as_float((c & 8u) << 28 | (c & 7u) << 22) * 0x1p126f) * scale;
  }
}

// Largest magnitude of 32 values (as bits: a NaN is larger than everything) -> scale code, and the factor that takes the values to E2M1's range:
// 2^(127 - code), 0 for a block that holds an infinity or a NaN (its codes are zeros).
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax_bits) {
  const int field = (int)(amax_bits >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - 2, 0);
}
__device__ __forceinline__ float mx_factor(uint32_t code) { return __uint_as_float((254u - code) << 23); }  // (code <= 252)
__device__ __forceinline__ float mx_scale(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7FC00000u : code == 0u ? 0x00400000u : code << 23);
}
__device__ __forceinline__ uint32_t mx_encode_block(float (&v)[8], uint32_t code) {
  if (code == 255u) return 0u;
  const float f = mx_factor(code);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= f;
  return mx_encode(v);
}

// byte of (row, block) in a scale tile of 128 rows x 4 blocks
__device__ __forceinline__ int mx_scale_at(int row, int blk) { return (row & 31) * 16 + (row >> 5) * 4 + blk; }

// A word of values: one fp32, or two bf16.  Largest magnitude as bits; value ``i`` of the 32 / sizeof(T) in 8 words; the other way.
template <typename T>
__device__ __forceinline__ uint32_t mx_word_max(uint32_t m, uint32_t u) {
  if constexpr (std::is_same<T, float>::value) return max(m, u & 0x7FFFFFFFu);
  else return __vmaxu2(m, u & 0x7FFF7FFFu);
}
template <typename T>
__device__ __forceinline__ uint32_t mx_word_max_bits(uint32_t m) {
  if constexpr (std::is_same<T, float>::value) return m;
  else return max(m & 0xFFFF0000u, m << 16);
}
template <typename T, int N>
__device__ __forceinline__ float mx_word_value(const uint32_t (&u)[N], int i) {
  if constexpr (std::is_same<T, float>::value) return __uint_as_float(u[i]);
  else return __uint_as_float(i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
}
template <typename T, int N>
__device__ __forceinline__ void mx_put(uint32_t (&u)[N], int i, T v) {  // (into zeros)
  if constexpr (std::is_same<T, float>::value) u[i] = __float_as_uint(v);
  else u[i / 2] |= (uint32_t)__bfloat16_as_ushort(v) << (16 * (i & 1));
}

// A stage of a product: 256 values of K, rows of 128 bytes, and the two scale tiles that lie along them
constexpr int MX_BK = 256, MX_ROW_BYTES = MX_BK / 2;
constexpr int MX_SCALE_TILE = 512, MX_STAGE_TILES = 2;
constexpr int MX_OP_BYTES = 128 * MX_ROW_BYTES;              // 128 rows of an operand
constexpr int MX_SC_BYTES = MX_STAGE_TILES * MX_SCALE_TILE;  // and their scales

__device__ __forceinline__ void st_32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}

// 32 columns of a row straight to C, in whole sectors; ``ncols`` of them lie in the matrix (whole sectors, too).
__device__ __forceinline__ void mx_store_row(uint8_t* dst, const uint32_t (&r)[32], int ncols, bool fp32) {
  if (fp32) {
#pragma unroll
    for (int j = 0; j < 32; j += 8)
      if (j < ncols) st_32(dst + 4 * j, r + j);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 16) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = pack_bf16(__uint_as_float(r[j + 2 * e]), __uint_as_float(r[j + 2 * e + 1]));
      if (j < ncols) st_32(dst + 2 * j, v);
    }
  }
}

// Epilogue of a warp's 32 rows and ``ncols`` columns (a multiple of 64), 32 at a time: from the first up, or ``down`` from the last; ``release`` as soon
// as the first 32 that way are in registers.  A load from TMEM takes some 400 cycles under load, so the next 32 columns are on their way while the
// last are stored.
template <typename Release>
__device__ __forceinline__ void mx_store_direct(const GemmParams& p, uint8_t* C, uint32_t taddr, int row0, int n0, int ncols, bool down, int lane,
                                                Release release) {
  const int esz = p.out_fp32 ? 4 : 2;
  const int chunks = ncols / 32, in = row0 + lane < p.M ? p.N - n0 : 0;  // columns of this row that lie in the matrix
  uint8_t* dst = C + ((row0 + lane) * p.ldc + n0) * esz;
  auto column = [&](int i) { return (down ? chunks - 1 - i : i) * 32; };
  uint32_t a[32], b[32];
  tmem_ld_32x32(taddr + column(0), a);
  tmem_ld_wait_for(a);
  release();
#pragma unroll 1
  for (int i = 0; i < chunks; i += 2) {
    tmem_ld_32x32(taddr + column(i + 1), b);
    mx_store_row(dst + column(i) * esz, a, in - column(i), p.out_fp32);
    tmem_ld_wait_for(b);
    const bool more = i + 2 < chunks;
    if (more) tmem_ld_32x32(taddr + column(i + 2), a);
    mx_store_row(dst + column(i + 1) * esz, b, in - column(i + 1), p.out_fp32);
    if (more) tmem_ld_wait_for(a);
  }
}

// [G][rows][bytes] of codes in boxes of 128 bytes x ``box_rows`` (128-byte swizzle), or [G][row tiles][scale words] in boxes of a stage's words.
inline int mx_map(CUtensorMap* m, const void* ptr, uint64_t inner, uint64_t rows, uint64_t G, uint32_t box_inner, uint32_t box_rows, bool scales) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return 1;
  const uint64_t esz = scales ? 4 : 1;
  cuuint64_t dims[3] = {inner, rows, G};
  cuuint64_t strides[2] = {inner * esz, inner * rows * esz};
  cuuint32_t box[3] = {box_inner, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, scales ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, scales ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 2;
}

}  // namespace apb
