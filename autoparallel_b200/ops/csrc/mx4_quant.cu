// Microscaled 4-bit floating point (MXFP4): quantisation, the values back, and both in one (formats and layout in ops/mx4_ops.py).
//
//   mx4_quantize    x [G, R, K] -> codes [G, R, Kp / 2], scales [G, R / 128, Kp / 128, 512]; x with unit stride along K, or along R
//   mx4_dequantize  the other way
//   mx4_round       x -> the values that its codes stand for, x's layout
//
// All are bound by memory: a CTA takes a tile of 128 rows x 128 columns, which is one scale tile, and reads and writes whole sectors of it.  A block's
// largest magnitude is an integer maximum of the values' bits, its scale a shift of them, the rounding the hardware's conversion (to nearest, ties to
// even), a value from its code the bits moved to an exponent and one multiplication.
// Measured for 64 x 1280 x 2048 bf16 (335 MB of values, 89 MB of codes), share of the copy rate: mx4_quantize 75 us (87 %), 64 x 2048 x 1408 with unit stride
// along the rows 80 (88 %), mx4_dequantize 75 to 80 (85 to 90 %), mx4_round 107 along K (96 %) and 117 to 128 along the rows.  Of 64 x 1279 x
// 2047, whose rows begin anywhere, hot: 89, 104 and 164 us, where 64 x 1280 x 2048 takes 67, 69 and 101; values of fp32, 16 x 695 x 1429: 16, 20 and 27.
// Compiled without --use_fast_math: denormals count.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mx4.cuh"

namespace apb {

constexpr int MX_THREADS = 256, MX_TILE = 128, MX_FEW_TILES = 4;

struct MxParams {
  const void *x, *x_end;  // (the byte after x's last value)
  uint8_t* codes;
  uint8_t* scales;
  void* y;
  long long G;
  int R, K, row_tiles, k_tiles, vec;
  long long gs, ld;  // elements of x between matrices and between rows (or columns, where the rows have unit stride)
};

// 32 bytes, where both the address and the row lengths allow it in one access (``wide``), otherwise in two.
__device__ __forceinline__ void load32(const void* p, bool wide, uint32_t (&u)[8]) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                 : "l"(p));
  } else {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w, u[4] = b.x, u[5] = b.y, u[6] = b.z, u[7] = b.w;
  }
}
__device__ __forceinline__ void store32(void* p, bool wide, const uint32_t (&u)[8]) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                 "r"(u[6]), "r"(u[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
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
// 32 bytes of a row (16 bf16 or 8 fp32, a half or a quarter of a block; the block's other threads are neighbours): the block's scale code, and the
// codes, or (``VALUES``) the values in place of what came in.
template <typename T, bool VALUES>
__device__ __forceinline__ uint32_t mx_round_32(uint32_t (&u)[8], uint32_t (&packed)[4 / (int)sizeof(T)]) {
  constexpr int PER = 32 / (int)sizeof(T);
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < 8; ++c) m = mx_word_max<T>(m, u[c]);
  uint32_t amax = mx_word_max_bits<T>(m);
#pragma unroll
  for (int d = 1; d < 32 / PER; d *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  const uint32_t code = mx_scale_code(amax);
#pragma unroll
  for (int h = 0; h < PER / 8; ++h) {
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = mx_word_value<T>(u, 8 * h + c);
    packed[h] = mx_encode_block(v, code);
    if (VALUES) {
      mx_decode(packed[h], mx_scale(code), v);
      if constexpr (PER == 8) {
#pragma unroll
        for (int c = 0; c < 8; ++c) u[c] = __float_as_uint(v[c]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) u[4 * h + c] = pack_bf16(v[2 * c], v[2 * c + 1]);
      }
    }
  }
  return code;
}
template <int PER>
__device__ __forceinline__ void mx_store_codes(const MxParams& p, const MxTile& at, int r, int k, int kp, const uint32_t (&packed)[PER / 8]) {
  if (r >= p.R || k >= kp) return;
  uint8_t* dst = p.codes + (at.g * p.R + r) * (kp / 2) + k / 2;
  if constexpr (PER == 16) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  else *reinterpret_cast<uint32_t*>(dst) = packed[0];
}

// Rows of 128 columns in shared memory, 16 bytes apart from the next but one's banks.
template <typename T>
constexpr int mx_pitch() { return MX_TILE * (int)sizeof(T) + 16; }

// 32 bytes of a row that begins anywhere, ``n`` of its values in the matrix: the 16-byte pieces of memory that have them, three at most, moved into place
// afterwards, so that several rows can be under way.  A piece may have values of the neighbours in memory, but none outside of x as a whole: the first and the last
// are put together value by value.  INSIDE: neither is among them; FULL: and all values are in the matrix.
template <typename T, bool INSIDE, bool FULL>
struct MxAnyRow {
  uint32_t w[12];
  uint32_t off;  // of the values in the pieces, bytes
  int n;
  __device__ __forceinline__ void load(const MxParams& p, const T* src, int count) {
    n = count;
    off = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15);
    const uint8_t* piece = reinterpret_cast<const uint8_t*>(src) - off;
#pragma unroll
    for (int q = 0; q < 3; ++q, piece += 16) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (FULL || (n > 0 && 16 * q < (int)off + n * (int)sizeof(T))) {
        if (INSIDE || (piece >= p.x && piece + 16 <= p.x_end)) v = *reinterpret_cast<const uint4*>(piece);
        else v = ends(p, piece);
      }
      w[4 * q] = v.x, w[4 * q + 1] = v.y, w[4 * q + 2] = v.z, w[4 * q + 3] = v.w;
    }
  }
  static __device__ __noinline__ uint4 ends(const MxParams& p, const uint8_t* piece) {
    uint32_t v[4] = {};
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      const T* at = reinterpret_cast<const T*>(piece) + i;
      if ((const void*)at >= p.x && (const void*)(at + 1) <= p.x_end) mx_put(v, i, *at);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ void words(uint32_t (&u)[8]) {
#pragma unroll
    for (int i = 0; i < 10; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 9; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
    constexpr int PER_WORD = 4 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = PER_WORD == 1 ? w[i] : __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
      if (!FULL) u[i] = i * PER_WORD >= n ? 0u : PER_WORD == 2 && i * PER_WORD + 1 >= n ? u[i] & 0xFFFFu : u[i];
    }
  }
};
template <typename T>
__device__ __forceinline__ void mx_row_out(T* dst, const T* row, int columns, int lane) {
#pragma unroll
  for (int c = 0; c < MX_TILE; c += 32)
    if (c + lane < columns) dst[c + lane] = row[c + lane];
}

// Unit stride along K, rows that are no whole 16 bytes.  Rounded values leave through shared memory, element by element but in whole sectors.  (Values that
// come in that way, too: 124 us for the codes of 64 x 1279 x 2047 bf16, 89 in 16-byte pieces; with the tests of the ends in every load 105.)
template <typename T, bool ROUND>
__global__ void __launch_bounds__(MX_THREADS) mx4_rows_any_kernel(MxParams p) {
  after_previous();
  constexpr int PER = 32 / (int)sizeof(T), ROW_THREADS = MX_TILE / PER, PASS = MX_THREADS / ROW_THREADS, ROWS = 2, CHUNK = ROWS * PASS;
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) uint8_t rows[ROUND ? CHUNK * mx_pitch<T>() : 16];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kp = (p.K + 31) / 32 * 32, columns = min(MX_TILE, p.K - at.k0);
  const int col = threadIdx.x % ROW_THREADS * PER, k = at.k0 + col, r_first = threadIdx.x / ROW_THREADS;
  const T* x = reinterpret_cast<const T*>(p.x) + at.g * p.gs + k;
  T* y = reinterpret_cast<T*>(p.y) + at.g * p.R * (long long)p.K + at.k0;
  auto run = [&](auto inside, auto full) {
#pragma unroll 1
    for (int r0 = 0; r0 < MX_TILE; r0 += CHUNK) {
      MxAnyRow<T, decltype(inside)::value, decltype(full)::value> in[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = at.r0 + r0 + r_first + PASS * i;
        in[i].load(p, x + r * p.ld, r < p.R ? min(PER, p.K - k) : 0);
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int rr = r0 + r_first + PASS * i, r = at.r0 + rr;
        uint32_t u[8], packed[PER / 8];
        in[i].words(u);
        const uint32_t code = mx_round_32<T, ROUND>(u, packed);
        if (ROUND) {
          uint4* own = reinterpret_cast<uint4*>(rows + (rr - r0) * mx_pitch<T>() + col * sizeof(T));
          own[0] = make_uint4(u[0], u[1], u[2], u[3]);
          own[1] = make_uint4(u[4], u[5], u[6], u[7]);
        } else {
          mx_store_codes<PER>(p, at, r, k, kp, packed);
          if (col % 32 == 0) tile[mx_scale_at(rr, col / 32)] = (uint8_t)(r < p.R && k < kp ? code : 127u);
        }
      }
      if (ROUND) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CHUNK / 8; ++i) {
          const int rr = warp + 8 * i, r = at.r0 + r0 + rr;
          if (r < p.R) mx_row_out(y + (long long)r * p.K, reinterpret_cast<const T*>(rows + rr * mx_pitch<T>()), columns, lane);
        }
        __syncthreads();
      }
    }
  };
  const uint8_t* first = reinterpret_cast<const uint8_t*>(x - col + at.r0 * p.ld);
  const uint8_t* end = reinterpret_cast<const uint8_t*>(x - col + (min(at.r0 + MX_TILE, p.R) - 1) * p.ld + MX_TILE);
  const bool inside = first - 15 >= p.x && end + 31 <= p.x_end;
  if (inside && at.r0 + MX_TILE <= p.R && at.k0 + MX_TILE <= p.K) run(std::true_type{}, std::true_type{});
  else if (inside) run(std::true_type{}, std::false_type{});
  else run(std::false_type{}, std::false_type{});
  if (!ROUND) {
    __syncthreads();
    if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(scale_tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(tile)[threadIdx.x];
  }
}

// Unit stride along K, rows of whole 16 bytes.  A thread has 32 bytes of a row (16 bf16 or 8 fp32), two or four threads a block; the loads of four rows are
// under way together.
// ROUND: the values in place of codes and scales.
template <typename T, bool ROUND>
__global__ void __launch_bounds__(MX_THREADS) mx4_rows_kernel(MxParams p) {
  after_previous();
  constexpr int PER = 32 / (int)sizeof(T), ROW_THREADS = MX_TILE / PER, PASS = MX_THREADS / ROW_THREADS, ROWS = 4;
  __shared__ __align__(16) uint8_t tile[512];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  const int kp = (p.K + 31) / 32 * 32, col = (threadIdx.x % ROW_THREADS) * PER, k = at.k0 + col, r_first = threadIdx.x / ROW_THREADS;
  const T* x = reinterpret_cast<const T*>(p.x) + at.g * p.gs;
#pragma unroll
  for (int pass = 0; pass < MX_TILE / PASS; pass += ROWS) {
    uint32_t u[ROWS][8];
    if (pass > 0 && at.r0 + pass * PASS >= p.R) {  // (whole passes without rows: only their scales are written)
      if (!ROUND && threadIdx.x < 128) {
        for (int i = threadIdx.x; i < (MX_TILE - pass * PASS) * 4; i += 128) tile[mx_scale_at(pass * PASS + i / 4, i & 3)] = 127;
      }
      break;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = at.r0 + r_first + PASS * (pass + i);
#pragma unroll
      for (int c = 0; c < 8; ++c) u[i][c] = 0;
      if (r < p.R) {
        const T* src = x + r * p.ld + k;
        if (k + PER <= p.K) {
          load32(src, p.vec > 1, u[i]);
        } else if (k < p.K) {  // (rows of whole 16 bytes)
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          u[i][0] = v.x, u[i][1] = v.y, u[i][2] = v.z, u[i][3] = v.w;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int rr = r_first + PASS * (pass + i), r = at.r0 + rr;
      const bool in = r < p.R && k < kp;
      uint32_t packed[PER / 8];
      const uint32_t code = mx_round_32<T, ROUND>(u[i], packed);
      if (ROUND) {
        T* dst = reinterpret_cast<T*>(p.y) + (at.g * p.R + r) * p.K + k;
        if (!in) continue;
        if (k + PER <= p.K) store32(dst, p.vec > 1, u[i]);
        else if (k < p.K) *reinterpret_cast<uint4*>(dst) = make_uint4(u[i][0], u[i][1], u[i][2], u[i][3]);
      } else {
        mx_store_codes<PER>(p, at, r, k, kp, packed);
        if (col % 32 == 0) tile[mx_scale_at(rr, col / 32)] = (uint8_t)(in ? code : 127u);
      }
    }
  }
  if (!ROUND) {
    __syncthreads();
    if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(scale_tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(tile)[threadIdx.x];
  }
}

// The codes of matrices with few rows, as many as a pass of the kernel above takes: four tiles that lie along K instead of four passes down one.  64 matrices of
// up to 32 rows of 2048: 2.9 to 3.3 us where a CTA for each tile takes 5.7 to 6.1 (1024 CTAs do not fit the chip at once); one of 17 x 14336 2.4 either way.
template <typename T>
__global__ void __launch_bounds__(MX_THREADS) mx4_few_rows_kernel(MxParams p) {
  after_previous();
  constexpr int PER = 32 / (int)sizeof(T), ROW_THREADS = MX_TILE / PER;
  __shared__ __align__(16) uint8_t tile[MX_FEW_TILES * 512];
  const int groups = (p.k_tiles + MX_FEW_TILES - 1) / MX_FEW_TILES, g = blockIdx.x / groups, kt = (blockIdx.x - g * groups) * MX_FEW_TILES;
  const MxTile at{g, 0, kt * MX_TILE};
  const int kp = (p.K + 31) / 32 * 32, col = threadIdx.x % ROW_THREADS * PER, r = threadIdx.x / ROW_THREADS;
  const T* row = reinterpret_cast<const T*>(p.x) + at.g * p.gs + r * p.ld;
  uint32_t u[MX_FEW_TILES][8];
#pragma unroll
  for (int i = 0; i < MX_FEW_TILES; ++i) {
    const int k = at.k0 + i * MX_TILE + col;
#pragma unroll
    for (int c = 0; c < 8; ++c) u[i][c] = 0;
    if (r >= p.R) continue;
    if (k + PER <= p.K) {
      load32(row + k, p.vec > 1, u[i]);
    } else if (k < p.K) {  // (rows of whole 16 bytes)
      const uint4 v = *reinterpret_cast<const uint4*>(row + k);
      u[i][0] = v.x, u[i][1] = v.y, u[i][2] = v.z, u[i][3] = v.w;
    }
  }
  static_assert(MX_FEW_TILES * 512 == MX_THREADS * 8, "eight bytes of the tiles a thread");
  reinterpret_cast<uint2*>(tile)[threadIdx.x] = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MX_FEW_TILES; ++i) {
    const int k = at.k0 + i * MX_TILE + col;
    uint32_t packed[PER / 8];
    const uint32_t code = mx_round_32<T, false>(u[i], packed);
    mx_store_codes<PER>(p, at, r, k, kp, packed);
    if (col % 32 == 0 && r < p.R && k < kp) tile[i * 512 + mx_scale_at(r, col / 32)] = (uint8_t)code;
  }
  __syncthreads();
  uint4* scales = reinterpret_cast<uint4*>(p.scales + ((long long)g * p.k_tiles + kt) * 512);
  if (threadIdx.x < min(MX_FEW_TILES, p.k_tiles - kt) * 32) scales[threadIdx.x] = reinterpret_cast<const uint4*>(tile)[threadIdx.x];
}

// Unit stride along R (a transposed matrix): a thread has a block of two neighbouring rows, and reads it column by column, a warp 64 rows at a time.
template <typename T, bool ROUND>
__global__ void __launch_bounds__(MX_THREADS) mx4_columns_kernel(MxParams p) {
  after_previous();
  constexpr int STRIDE = 80;  // bytes of a row of codes in shared memory (64 used)
  constexpr int W = 2 * (int)sizeof(T) / 4;  // words of two rows in a column
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) uint8_t rows[ROUND ? 16 : MX_TILE * STRIDE];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  const int kp = (p.K + 31) / 32 * 32, rr = (threadIdx.x & 63) * 2, r = at.r0 + rr, blk = threadIdx.x >> 6, k = at.k0 + blk * 32;
  const T* x = reinterpret_cast<const T*>(p.x) + at.g * p.gs + r;
  uint32_t u[32][W];
  const bool whole = p.vec && k + 32 <= p.K && r < p.R;
  if (!p.vec && k + 32 <= p.K && r + 1 < p.R) {  // (a column begins anywhere)
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const T* src = x + (long long)(k + i) * p.ld;
      if constexpr (W == 2) {
        u[i][0] = __float_as_uint(src[0]);
        u[i][1] = __float_as_uint(src[1]);
      } else {
        u[i][0] = __bfloat16_as_ushort(src[0]) | (uint32_t)__bfloat16_as_ushort(src[1]) << 16;
      }
    }
  } else if (whole) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const T* src = x + (long long)(k + i) * p.ld;
      if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        u[i][0] = v.x, u[i][1] = v.y;
      } else {
        u[i][0] = *reinterpret_cast<const uint32_t*>(src);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const T* src = x + (long long)(k + i) * p.ld;
#pragma unroll
      for (int w = 0; w < W; ++w) u[i][w] = 0;
      if (k + i < p.K) {
        if constexpr (W == 2) {
          if (r < p.R) u[i][0] = __float_as_uint(src[0]);
          if (r + 1 < p.R) u[i][1] = __float_as_uint(src[1]);
        } else {
          if (r < p.R) u[i][0] = __bfloat16_as_ushort(src[0]);
          if (r + 1 < p.R) u[i][0] |= (uint32_t)__bfloat16_as_ushort(src[1]) << 16;
        }
      }
    }
  }
  uint32_t m[W] = {};
#pragma unroll
  for (int i = 0; i < 32; ++i)
#pragma unroll
    for (int w = 0; w < W; ++w) m[w] = mx_word_max<T>(m[w], u[i][w]);
  uint32_t code[2], packed[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    code[h] = mx_scale_code(W == 2 ? m[W == 2 ? h : 0] : h == 0 ? m[0] << 16 : m[0] & 0xFFFF0000u);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx_word_value<T>(u[8 * q + i], h);
      packed[h][q] = mx_encode_block(v, code[h]);
    }
  }
  if (ROUND) {
    T* y = reinterpret_cast<T*>(p.y) + at.g * p.R * p.K + r;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float a[8], b[8];
      mx_decode(packed[0][q], mx_scale(code[0]), a);
      mx_decode(packed[1][q], mx_scale(code[1]), b);
      if (whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          T* dst = y + (long long)(k + 8 * q + i) * p.R;
          if constexpr (W == 2) *reinterpret_cast<float2*>(dst) = make_float2(a[i], b[i]);
          else *reinterpret_cast<uint32_t*>(dst) = pack_bf16(a[i], b[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          T* dst = y + (long long)(k + 8 * q + i) * p.R;
          if (k + 8 * q + i < p.K && r < p.R) store1(dst, a[i]);
          if (k + 8 * q + i < p.K && r + 1 < p.R) store1(dst + 1, b[i]);
        }
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<uint4*>(rows + (rr + h) * STRIDE + blk * 16) = make_uint4(packed[h][0], packed[h][1], packed[h][2], packed[h][3]);
      tile[mx_scale_at(rr + h, blk)] = (uint8_t)(r + h < p.R && k < kp ? code[h] : 127u);
    }
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

// A thread has 16 values of a row: 8 bytes of codes, all its rows under way together.  STAGED: rows that are no whole 16 bytes leave through shared
// memory, element by element but in whole sectors.
template <typename T, bool STAGED>
__global__ void __launch_bounds__(MX_THREADS) mx4_dequantize_kernel(MxParams p) {
  after_previous();
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) uint8_t rows[STAGED ? 32 * mx_pitch<T>() : 16];
  uint8_t* scale_tile = nullptr;
  const MxTile at = mx_tile(p, &scale_tile);
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(tile)[threadIdx.x] = reinterpret_cast<const uint32_t*>(scale_tile)[threadIdx.x];
  const int kp = (p.K + 31) / 32 * 32, col = (threadIdx.x & 7) * 16, k = at.k0 + col, r_first = threadIdx.x >> 3;
  uint2 packed[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = at.r0 + r_first + 32 * i;
    packed[i] = make_uint2(0, 0);
    if (r < p.R && k < p.K) packed[i] = *reinterpret_cast<const uint2*>(p.codes + (at.g * p.R + r) * (kp / 2) + k / 2);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = r_first + 32 * i, r = at.r0 + rr;
    constexpr int PER = 32 / (int)sizeof(T);
    float v[16];
    const float scale = mx_scale(tile[mx_scale_at(rr, col / 32)]);
    float (&lo)[8] = *reinterpret_cast<float (*)[8]>(v), (&hi)[8] = *reinterpret_cast<float (*)[8]>(v + 8);
    mx_decode(packed[i].x, scale, lo);
    mx_decode(packed[i].y, scale, hi);
    uint32_t u[16 / PER][8];
#pragma unroll
    for (int h = 0; h < 16 / PER; ++h)
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if constexpr (PER == 8) u[h][c] = __float_as_uint(v[8 * h + c]);
        else u[h][c] = pack_bf16(v[2 * c], v[2 * c + 1]);
      }
    if (STAGED) {
      uint4* own = reinterpret_cast<uint4*>(rows + r_first * mx_pitch<T>() + col * sizeof(T));
#pragma unroll
      for (int h = 0; h < 16 / PER; ++h) {
        own[2 * h] = make_uint4(u[h][0], u[h][1], u[h][2], u[h][3]);
        own[2 * h + 1] = make_uint4(u[h][4], u[h][5], u[h][6], u[h][7]);
      }
      __syncthreads();
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int out = at.r0 + 32 * i + warp + 8 * j;
        if (out < p.R)
          mx_row_out(reinterpret_cast<T*>(p.y) + (at.g * p.R + out) * (long long)p.K + at.k0, reinterpret_cast<const T*>(rows + (warp + 8 * j) * mx_pitch<T>()),
                     min(MX_TILE, p.K - at.k0), lane);
      }
      __syncthreads();
    } else if (r < p.R && k < p.K) {
      T* dst = reinterpret_cast<T*>(p.y) + (at.g * p.R + r) * p.K + k;
#pragma unroll
      for (int h = 0; h < 16 / PER; ++h) {
        if (k + PER * (h + 1) <= p.K) store32(dst + PER * h, p.vec > 1, u[h]);
        else if (k + PER * h < p.K) *reinterpret_cast<uint4*>(dst + PER * h) = make_uint4(u[h][0], u[h][1], u[h][2], u[h][3]);  // (rows of whole 16 bytes)
      }
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
    // rows that begin on 32 or on 16 bytes, and end there (so do those of the result)
    auto whole = [&](int bytes) {
      return p.ld * esz % bytes == 0 && p.gs * esz % bytes == 0 && (long long)p.K * esz % bytes == 0 && aligned(p.x, bytes) && (!ROUND || aligned(p.y, bytes));
    };
    p.vec = whole(32) ? 2 : whole(16) ? 1 : 0;
    p.x_end = reinterpret_cast<const uint8_t*>(p.x) + ((p.G - 1) * p.gs + (p.R - 1) * p.ld + p.K) * esz;
    if (!ROUND && p.vec && p.R <= MX_THREADS * (32 / esz) / MX_TILE) {
      const unsigned few = (unsigned)(p.G * ((p.k_tiles + MX_FEW_TILES - 1) / MX_FEW_TILES));
      is_bf16 ? launch_after(mx4_few_rows_kernel<__nv_bfloat16>, few, MX_THREADS, 0, st, p) : launch_after(mx4_few_rows_kernel<float>, few, MX_THREADS, 0, st, p);
    } else if (p.vec)
      is_bf16 ? launch_after(mx4_rows_kernel<__nv_bfloat16, ROUND>, grid, MX_THREADS, 0, st, p)
              : launch_after(mx4_rows_kernel<float, ROUND>, grid, MX_THREADS, 0, st, p);
    else
      is_bf16 ? launch_after(mx4_rows_any_kernel<__nv_bfloat16, ROUND>, grid, MX_THREADS, 0, st, p)
              : launch_after(mx4_rows_any_kernel<float, ROUND>, grid, MX_THREADS, 0, st, p);
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
  const int esz = is_bf16 ? 2 : 4;
  p.vec = K * esz % 32 == 0 && aligned(y, 32) ? 2 : K * esz % 16 == 0 ? 1 : 0;
  if (p.vec)
    is_bf16 ? launch_after(mx4_dequantize_kernel<__nv_bfloat16, false>, grid, MX_THREADS, 0, st, p)
            : launch_after(mx4_dequantize_kernel<float, false>, grid, MX_THREADS, 0, st, p);
  else
    is_bf16 ? launch_after(mx4_dequantize_kernel<__nv_bfloat16, true>, grid, MX_THREADS, 0, st, p)
            : launch_after(mx4_dequantize_kernel<float, true>, grid, MX_THREADS, 0, st, p);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
