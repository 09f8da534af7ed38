// Activations to 8 bits and back (mx8.cuh), and the middle of a gated feed-forward block element by element (gated.cuh) for operands that the products of
// gemm_gated.cu do not take.  All are bound by memory.
#include "rowwise.cuh"

#include "gated.cuh"

namespace apb {

typedef __nv_bfloat16 bf16;

// Rows of whole blocks lie one behind the other, so the matrix is one row of blocks: sixteen elements to a thread, two threads to a block, the codes of a
// thread are one vector.
template <typename T>
__global__ void __launch_bounds__(256) mx8_quantize_kernel(const T* x, uint8_t* codes, uint8_t* scales, long long n16) {
  after_previous();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  const bool in = i < n16;  // (both threads of a block are in or out)
  Vec8<T> lo, hi;
  float f[16], g[8];
  uint32_t top = 0;
  if (in) {
    lo.load(x + i * 16);
    hi.load(x + i * 16 + 8);
    lo.to_float(g);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = g[k];
    hi.to_float(g);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[8 + k] = g[k];
#pragma unroll
    for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(f[k]) & 0x7fffffffu);
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  if (!in) return;
  const uint32_t byte = mx8_scale_byte(top);
  const Mx8Coder coder(byte, top);
  auto four = [&](int k) { return coder.four(__float_as_uint(f[k]), __float_as_uint(f[k + 1]), __float_as_uint(f[k + 2]), __float_as_uint(f[k + 3])); };
  reinterpret_cast<uint4*>(codes)[i] = make_uint4(four(0), four(4), four(8), four(12));
  if ((i & 1) == 0) scales[i >> 1] = (uint8_t)byte;
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* y, long long n16) {
  after_previous();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n16) return;
  const uint4 c = reinterpret_cast<const uint4*>(codes)[i];
  const Mx8Reader reader(scales[i >> 1]);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[8];
    reader.four(w[2 * h], f);
    reader.four(w[2 * h + 1], f + 4);
    Vec8<T> o;
    o.from_float(f);
    o.store(y + i * 16 + 8 * h);
  }
}

// Rows whose last block is not full begin anywhere: a warp to a block, an element to a lane, RAGGED blocks of a row under way together.
constexpr int RAGGED = 4;
template <typename T>
__global__ void __launch_bounds__(256) mx8_quantize_ragged_kernel(const T* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int blocks, int groups) {
  after_previous();
  const long long w = blockIdx.x * 8ll + (threadIdx.x >> 5);  // (a warp: RAGGED blocks of one row)
  const int lane = threadIdx.x & 31;
  const long long row = w / groups;
  if (row >= rows) return;
  const int b0 = (int)(w - row * groups) * RAGGED;
  float v[RAGGED];
#pragma unroll
  for (int j = 0; j < RAGGED; ++j) {
    const int c = (b0 + j) * MX8_BLOCK + lane;
    v[j] = c < K ? float(x[row * K + c]) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < RAGGED; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7fffffffu), byte = mx8_scale_byte(top);
    const int c = (b0 + j) * MX8_BLOCK + lane;
    if (c < K) codes[row * K + c] = (uint8_t)Mx8Coder(byte, top).four(__float_as_uint(v[j]), 0, 0, 0);
    if (lane == 0 && b0 + j < blocks) scales[row * blocks + b0 + j] = (uint8_t)byte;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_ragged_kernel(const uint8_t* codes, const uint8_t* scales, T* y, long long rows, int K, int blocks,
                                                                   int groups) {
  after_previous();
  const long long w = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long row = w / groups;
  if (row >= rows) return;
  const int b0 = (int)(w - row * groups) * RAGGED;
  uint32_t code[RAGGED], byte[RAGGED];
#pragma unroll
  for (int j = 0; j < RAGGED; ++j) {
    const int c = (b0 + j) * MX8_BLOCK + lane;
    if (c < K) {
      code[j] = codes[row * K + c];
      byte[j] = scales[row * blocks + b0 + j];
    }
  }
#pragma unroll
  for (int j = 0; j < RAGGED; ++j) {
    const int c = (b0 + j) * MX8_BLOCK + lane;
    if (c < K) {
      float f[4];
      Mx8Reader(byte[j]).four(code[j], f);
      y[row * K + c] = T(f[0]);
    }
  }
}

// ab fp32 [M, 2, H] -> h [M, H]; and dh fp32 [M, H] with ab -> dab [M, 2, H], h
template <typename T>
__global__ void __launch_bounds__(256) gated_act_kernel(const float* ab, T* h, long long n, int H, int act) {
  after_previous();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long row = i / H;
  const float a = ab[i + row * H], b = ab[i + row * H + H];
  with_act(act, [&](auto k) {
    float d;
    h[i] = T(act_value<decltype(k)::value, true>(a, d) * b);
  });
}
template <typename T>
__global__ void __launch_bounds__(256) gated_act_bwd_kernel(const float* dh, const float* ab, T* dab, T* h, long long n, int H, int act) {
  after_previous();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long at = i + i / H * H;
  float da, db, v;
  with_act(act, [&](auto k) { gated_grad<decltype(k)::value, true>(dh[i], ab[at], ab[at + H], da, db, v); });
  dab[at] = T(da);
  dab[at + H] = T(db);
  h[i] = T(v);
}

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
static int done(cudaError_t e) { return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4; }
// blocks of 256 threads for n of them; 0: more than a launch has
static unsigned blocks_of(long long n) { return (n + 255) / 256 > 0x7fffffffll ? 0u : (unsigned)((n + 255) / 256); }

}  // namespace apb

using namespace apb;

// x [R, K], codes [R, K], scales [R, ceil(K / 32)], all dense, x and codes on 16-byte bases.
extern "C" int apb_mx8_quantize(const void* x, void* codes, void* scales, long long R, long long K, int is_bf16, cudaStream_t st) {
  if (R <= 0 || K <= 0) return 0;
  if (off16(x) || off16(codes) || K > 0x7fffffe0ll) return 3;
  uint8_t *c = (uint8_t*)codes, *s = (uint8_t*)scales;
  const long long blocks = (K + MX8_BLOCK - 1) / MX8_BLOCK, groups = (blocks + RAGGED - 1) / RAGGED;
  const unsigned grid = blocks_of(K % MX8_BLOCK == 0 ? R * K / 16 : R * groups * 32);
  if (grid == 0) return 3;
  if (K % MX8_BLOCK == 0)
    return done(is_bf16 ? launch_after(mx8_quantize_kernel<bf16>, grid, 256, 0, st, (const bf16*)x, c, s, R * K / 16)
                        : launch_after(mx8_quantize_kernel<float>, grid, 256, 0, st, (const float*)x, c, s, R * K / 16));
  return done(is_bf16 ? launch_after(mx8_quantize_ragged_kernel<bf16>, grid, 256, 0, st, (const bf16*)x, c, s, R, (int)K, (int)blocks, (int)groups)
                      : launch_after(mx8_quantize_ragged_kernel<float>, grid, 256, 0, st, (const float*)x, c, s, R, (int)K, (int)blocks, (int)groups));
}
extern "C" int apb_mx8_dequantize(const void* codes, const void* scales, void* y, long long R, long long K, int is_bf16, cudaStream_t st) {
  if (R <= 0 || K <= 0) return 0;
  if (off16(y) || off16(codes) || K > 0x7fffffe0ll) return 3;
  const uint8_t *c = (const uint8_t*)codes, *s = (const uint8_t*)scales;
  const long long blocks = (K + MX8_BLOCK - 1) / MX8_BLOCK, groups = (blocks + RAGGED - 1) / RAGGED;
  const unsigned grid = blocks_of(K % MX8_BLOCK == 0 ? R * K / 16 : R * groups * 32);
  if (grid == 0) return 3;
  if (K % MX8_BLOCK == 0)
    return done(is_bf16 ? launch_after(mx8_dequantize_kernel<bf16>, grid, 256, 0, st, c, s, (bf16*)y, R * K / 16)
                        : launch_after(mx8_dequantize_kernel<float>, grid, 256, 0, st, c, s, (float*)y, R * K / 16));
  return done(is_bf16 ? launch_after(mx8_dequantize_ragged_kernel<bf16>, grid, 256, 0, st, c, s, (bf16*)y, R, (int)K, (int)blocks, (int)groups)
                      : launch_after(mx8_dequantize_ragged_kernel<float>, grid, 256, 0, st, c, s, (float*)y, R, (int)K, (int)blocks, (int)groups));
}

extern "C" int apb_gated_act(const float* ab, void* h, long long M, int H, int act, int is_bf16, cudaStream_t st) {
  if (M <= 0 || H <= 0) return 0;
  const unsigned grid = blocks_of(M * H);
  if (grid == 0) return 3;
  return done(is_bf16 ? launch_after(gated_act_kernel<bf16>, grid, 256, 0, st, ab, (bf16*)h, M * H, H, act)
                      : launch_after(gated_act_kernel<float>, grid, 256, 0, st, ab, (float*)h, M * H, H, act));
}
extern "C" int apb_gated_act_bwd(const float* dh, const float* ab, void* dab, void* h, long long M, int H, int act, int is_bf16, cudaStream_t st) {
  if (M <= 0 || H <= 0) return 0;
  const unsigned grid = blocks_of(M * H);
  if (grid == 0) return 3;
  return done(is_bf16 ? launch_after(gated_act_bwd_kernel<bf16>, grid, 256, 0, st, dh, ab, (bf16*)dab, (bf16*)h, M * H, H, act)
                      : launch_after(gated_act_bwd_kernel<float>, grid, 256, 0, st, dh, ab, (float*)dab, (float*)h, M * H, H, act));
}
