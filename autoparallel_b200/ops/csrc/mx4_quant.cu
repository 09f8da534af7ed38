// Microscaled 4-bit floating point (MXFP4): quantisation, the values back, and both in one (formats and layout in ops/mx4_ops.py).
//
//   mx4_quantize    x [G, R, K] -> codes [G, R, Kp / 2], scales [G, R / 128, Kp / 128, 512]; x with unit stride along K, or along R
//   mx4_dequantize  the other way
//   mx4_round       x -> the values that its codes stand for, x's layout
//
// All are bound by memory: a CTA takes a tile of 128 rows x 128 columns, which is one scale tile, and reads and writes whole sectors of it.
// Compiled without --use_fast_math: denormals count.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.cuh"

namespace apb {

constexpr int MX_THREADS = 256, MX_TILE = 128;

struct MxParams {
  const void* x;
  uint8_t* codes;
  uint8_t* scales;
  void* y;
  long long G;
  int R, K, row_tiles, k_tiles, vec;
  long long gs, ld;  // elements of x between matrices and between rows (or columns, where the rows have unit stride)
};

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

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
template <typename T>
__device__ __forceinline__ float mx_load(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *p;
  else return __bfloat162float(*p);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4);
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <typename T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (std::is_same<T, float>::value) *p = v;
  else *p = __float2bfloat16(v);
}

struct MxTile {
  long long g;
  int r0, k0;
};
__device__ __forceinline__ MxTile mx_tile(const MxParams& p, uint8_t** scale_tile) {
  const long long t = blockIdx.x;
  const int kt = (int)(t % p.k_tiles);
  const long long rest = t / p.k_tiles;
  const int rt = (int)(rest % p.row_tiles);
  if (p.scales != nullptr) *scale_tile = p.scales + t * 512;  // (tiles lie in the order of the grid)
  return {rest / p.row_tiles, rt * MX_TILE, kt * MX_TILE};
}
// byte of (row, block) in a scale tile
__device__ __forceinline__ int scale_at(int row, int blk) { return (row & 31) * 16 + (row >> 5) * 4 + blk; }

// Unit stride along K.  A thread has 8 columns of a row, four threads a block, 16 a row of the tile; all its rows are loaded before the first is used.
// ROUND: the values in place of codes and scales.
template <typename T, bool ROUND>
__global__ void __launch_bounds__(MX_THREADS) mx4_rows_kernel(MxParams p) {
  after_previous();
  __shared__ __align__(16) uint8_t tile[512];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  const int kp = (p.K + 31) / 32 * 32, col = (threadIdx.x & 15) * 8, k = at.k0 + col, r_first = threadIdx.x >> 4;
  const T* x = reinterpret_cast<const T*>(p.x) + at.g * p.gs;
  constexpr int ROWS = 4;  // under way together
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float v[ROWS][8];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = at.r0 + r_first + 16 * (ROWS * half + i);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[i][c] = 0.f;
      if (r < p.R) {
        const T* src = x + r * p.ld + k;
        if (p.vec) {
          if (k < p.K) load8(src, v[i]);
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (k + c < p.K) v[i][c] = mx_load(src + c);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int rr = r_first + 16 * (ROWS * half + i), r = at.r0 + rr;
      uint32_t amax = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) amax = max(amax, abs_bits(v[i][c]));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const uint32_t code = mx_scale_code(amax);
      const uint32_t packed = mx_encode_block(v[i], code);
      const bool in = r < p.R && k < kp;
      if (ROUND) {
        if (in) {
          mx_decode(packed, mx_scale(code), v[i]);
          T* dst = reinterpret_cast<T*>(p.y) + (at.g * p.R + r) * p.K + k;
          if (p.vec) {
            if (k < p.K) store8(dst, v[i]);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              if (k + c < p.K) store1(dst + c, v[i][c]);
          }
        }
      } else {
        if (in) *reinterpret_cast<uint32_t*>(p.codes + (at.g * p.R + r) * (kp / 2) + k / 2) = packed;
        if ((threadIdx.x & 3) == 0) tile[scale_at(rr, col / 32)] = (uint8_t)(in ? code : 127u);
      }
    }
  }
  if (!ROUND) {
    __syncthreads();
    if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(scale_tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(tile)[threadIdx.x];
  }
}

// Unit stride along R (a transposed matrix): a thread has a block of two neighbouring rows, and reads it column by column, a warp 64 rows at a time.
template <typename T, bool ROUND>
__global__ void __launch_bounds__(MX_THREADS) mx4_columns_kernel(MxParams p) {
  after_previous();
  constexpr int STRIDE = 80;  // bytes of a row of codes in shared memory (64 used)
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) uint8_t rows[ROUND ? 16 : MX_TILE * STRIDE];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  const int kp = (p.K + 31) / 32 * 32, rr = (threadIdx.x & 63) * 2, r = at.r0 + rr, blk = threadIdx.x >> 6, k = at.k0 + blk * 32;
  const T* x = reinterpret_cast<const T*>(p.x) + at.g * p.gs + r;
  float v[2][32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[0][i] = v[1][i] = 0.f;
    if (k + i < p.K) {
      const T* src = x + (k + i) * p.ld;
      if (p.vec) {
        if (r < p.R) {
          if constexpr (std::is_same<T, float>::value) {
            const float2 f = *reinterpret_cast<const float2*>(src);
            v[0][i] = f.x;
            v[1][i] = f.y;
          } else {
            const uint32_t u = *reinterpret_cast<const uint32_t*>(src);
            v[0][i] = __uint_as_float(u << 16);
            v[1][i] = __uint_as_float(u & 0xFFFF0000u);
          }
        }
      } else {
        if (r < p.R) v[0][i] = mx_load(src);
        if (r + 1 < p.R) v[1][i] = mx_load(src + 1);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, abs_bits(v[h][i]));
    const uint32_t code = mx_scale_code(amax);
    uint32_t packed[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = v[h][8 * q + i];
      packed[q] = mx_encode_block(w, code);
      if (ROUND) {
        mx_decode(packed[q], mx_scale(code), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h][8 * q + i] = w[i];
      }
    }
    if (!ROUND) {
      *reinterpret_cast<uint4*>(rows + (rr + h) * STRIDE + blk * 16) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      tile[scale_at(rr + h, blk)] = (uint8_t)(r + h < p.R && k < kp ? code : 127u);
    }
  }
  if (ROUND) {
    T* y = reinterpret_cast<T*>(p.y) + at.g * p.R * p.K + r;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (k + i >= p.K) break;
      T* dst = y + (long long)(k + i) * p.R;
      if (p.vec) {
        if (r < p.R) {
          if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float2*>(dst) = make_float2(v[0][i], v[1][i]);
          else *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(v[0][i], v[1][i]);
        }
      } else {
        if (r < p.R) store1(dst, v[0][i]);
        if (r + 1 < p.R) store1(dst + 1, v[1][i]);
      }
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = (threadIdx.x >> 2) + 64 * h, c = threadIdx.x & 3;
      if (at.r0 + row < p.R && at.k0 + c * 32 < kp)
        *reinterpret_cast<uint4*>(p.codes + (at.g * p.R + at.r0 + row) * (kp / 2) + at.k0 / 2 + c * 16) =
            *reinterpret_cast<const uint4*>(rows + row * STRIDE + c * 16);
    }
    if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(scale_tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(tile)[threadIdx.x];
  }
}

template <typename T>
__global__ void __launch_bounds__(MX_THREADS) mx4_dequantize_kernel(MxParams p) {
  after_previous();
  __shared__ __align__(16) uint8_t tile[512];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(scale_tile)[threadIdx.x];
  const int kp = (p.K + 31) / 32 * 32, col = (threadIdx.x & 15) * 8, k = at.k0 + col, r_first = threadIdx.x >> 4;
  uint32_t packed[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = at.r0 + r_first + 16 * i;
    packed[i] = 0;
    if (r < p.R && k < p.K) packed[i] = *reinterpret_cast<const uint32_t*>(p.codes + (at.g * p.R + r) * (kp / 2) + k / 2);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rr = r_first + 16 * i, r = at.r0 + rr;
    if (r >= p.R || k >= p.K) continue;
    float v[8];
    mx_decode(packed[i], mx_scale(tile[scale_at(rr, col / 32)]), v);
    T* dst = reinterpret_cast<T*>(p.y) + (at.g * p.R + r) * p.K + k;
    if (p.vec) {
      store8(dst, v);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (k + c < p.K) store1(dst + c, v[c]);
    }
  }
}

static bool mx_grid(MxParams& p, long long G, long long R, long long K, unsigned* grid) {
  if (G < 0 || R < 0 || K < 0 || R >= 1ll << 31 || K >= 1ll << 30) return false;
  p.G = G;
  p.R = (int)R;
  p.K = (int)K;
  p.row_tiles = (int)((R + MX_TILE - 1) / MX_TILE);
  p.k_tiles = (int)((K + MX_TILE - 1) / MX_TILE);
  const long long tiles = G * p.row_tiles * p.k_tiles;
  if (tiles >= 1ll << 31) return false;
  *grid = (unsigned)tiles;
  return true;
}
static bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <bool ROUND>
static int mx_from_values(MxParams& p, unsigned grid, int transposed, int is_bf16, cudaStream_t st) {
  if (grid == 0) return 0;
  const int esz = is_bf16 ? 2 : 4;
  if (transposed) {
    p.vec = p.ld % 2 == 0 && p.gs % 2 == 0 && p.R % 2 == 0 && aligned(p.x, 2 * esz);
    is_bf16 ? launch_after(mx4_columns_kernel<__nv_bfloat16, ROUND>, grid, MX_THREADS, 0, st, p)
            : launch_after(mx4_columns_kernel<float, ROUND>, grid, MX_THREADS, 0, st, p);
  } else {
    p.vec = p.ld * esz % 16 == 0 && p.gs * esz % 16 == 0 && p.K % 8 == 0 && aligned(p.x, 16);
    is_bf16 ? launch_after(mx4_rows_kernel<__nv_bfloat16, ROUND>, grid, MX_THREADS, 0, st, p)
            : launch_after(mx4_rows_kernel<float, ROUND>, grid, MX_THREADS, 0, st, p);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace apb

using namespace apb;

// x: element (g, r, k) at g * gs + r * ld + k, or at g * gs + k * ld + r if ``transposed``; codes, scales dense with 16-byte bases.
// Return 0, or an argument / launch error (nothing launched).
extern "C" int apb_mx4_quantize(const void* x, void* codes, void* scales, long long G, long long R, long long K, long long gs, long long ld,
                                int transposed, int is_bf16, cudaStream_t st) {
  MxParams p{};
  unsigned grid = 0;
  if (!mx_grid(p, G, R, K, &grid) || !aligned(codes, 16) || !aligned(scales, 16)) return 3;
  p.x = x;
  p.codes = (uint8_t*)codes;
  p.scales = (uint8_t*)scales;
  p.gs = gs;
  p.ld = ld;
  return mx_from_values<false>(p, grid, transposed, is_bf16, st);
}

// y: [G, R, K], or [G, K, R] if ``transposed``, dense with a 16-byte base.
extern "C" int apb_mx4_round(const void* x, void* y, long long G, long long R, long long K, long long gs, long long ld, int transposed, int is_bf16,
                             cudaStream_t st) {
  MxParams p{};
  unsigned grid = 0;
  if (!mx_grid(p, G, R, K, &grid) || !aligned(y, 16)) return 3;
  p.x = x;
  p.y = y;
  p.gs = gs;
  p.ld = ld;
  return mx_from_values<true>(p, grid, transposed, is_bf16, st);
}

extern "C" int apb_mx4_dequantize(const void* codes, const void* scales, void* y, long long G, long long R, long long K, int is_bf16, cudaStream_t st) {
  MxParams p{};
  unsigned grid = 0;
  if (!mx_grid(p, G, R, K, &grid) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(y, 16)) return 3;
  if (grid == 0) return 0;
  p.codes = (uint8_t*)const_cast<void*>(codes);
  p.scales = (uint8_t*)const_cast<void*>(scales);
  p.y = y;
  p.vec = K % 8 == 0;
  is_bf16 ? launch_after(mx4_dequantize_kernel<__nv_bfloat16>, grid, MX_THREADS, 0, st, p)
          : launch_after(mx4_dequantize_kernel<float>, grid, MX_THREADS, 0, st, p);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
