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
  const uint32_t byte = mx_scale_byte<8>(top);
  const MxCoder<8> coder(byte, top);
  uint32_t u[16], c[4];
#pragma unroll
  for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(f[k]);
  coder.words(u, c);
  reinterpret_cast<uint4*>(codes)[i] = make_uint4(c[0], c[1], c[2], c[3]);
  if ((i & 1) == 0) scales[i >> 1] = (uint8_t)byte;
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* y, long long n16) {
  after_previous();
  if constexpr (sizeof(T) == 4) {
    // sixteen fp32 values of a thread would be pieces of 16 bytes in every line that a warp stores; four times four, a warp's width apart, are whole lines
    // (8192 x 4096 38.9 -> 28.4 us)
    const long long first = (blockIdx.x * 256ll + (threadIdx.x & ~31)) * 4 + (threadIdx.x & 31);  // (in pieces of four)
    uint32_t c[4];
    uint8_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long i = first + 32 * k;
      if (i < n16 * 4) {
        c[k] = reinterpret_cast<const uint32_t*>(codes)[i];
        b[k] = scales[i >> 3];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long i = first + 32 * k;
      float f[4];
      MxReader<8>(b[k]).four(c[k], f);
      if (i < n16 * 4) reinterpret_cast<float4*>(y)[i] = make_float4(f[0], f[1], f[2], f[3]);
    }
    return;
  }
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n16) return;
  const uint4 c = reinterpret_cast<const uint4*>(codes)[i];
  const MxReader<8> reader(scales[i >> 1]);
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

// Rows of whole vectors whose last block is not full: eight elements to a thread, four threads to a block, ``vecs`` threads (four to every block) to a row.
template <typename T>
__global__ void __launch_bounds__(256) mx8_quantize_vec_kernel(const T* x, uint8_t* codes, uint8_t* scales, uint32_t rows, int K, uint32_t vecs) {
  after_previous();
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, row = i / vecs, c = (i - row * vecs) * 8;
  const bool in = row < rows && c < (uint32_t)K;
  const long long e = (long long)row * K + c;
  float f[8] = {};
  if (in) {
    Vec8<T> v;
    v.load(x + e);
    v.to_float(f);
  }
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(f[k]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (!in) return;
  const uint32_t byte = mx_scale_byte<8>(top);
  const MxCoder<8> coder(byte, top);
  uint32_t u[8], w[2];
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = __float_as_uint(f[k]);
  coder.words(u, w);
  *reinterpret_cast<uint2*>(codes + e) = make_uint2(w[0], w[1]);
  if (c % MX_BLOCK == 0) scales[(long long)row * (vecs / 4) + c / MX_BLOCK] = (uint8_t)byte;
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_vec_kernel(const uint8_t* codes, const uint8_t* scales, T* y, uint32_t rows, int K, uint32_t vecs) {
  after_previous();
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, row = i / vecs, c = (i - row * vecs) * 8;
  if (row >= rows || c >= (uint32_t)K) return;
  const long long e = (long long)row * K + c;
  const uint2 w = *reinterpret_cast<const uint2*>(codes + e);
  const MxReader<8> reader(scales[(long long)row * (vecs / 4) + c / MX_BLOCK]);
  float f[8];
  reader.four(w.x, f);
  reader.four(w.y, f + 4);
  Vec8<T> o;
  o.from_float(f);
  o.store(y + e);
}

// Other rows begin anywhere.  A warp has seven blocks of a row, 224 elements, and takes them in the tensor's own aligned vectors of
// eight elements (at most 29 of them, one to a lane): a lane's elements belong to one block or to two neighbours, ``first`` and the one after.  Codes lie like
// the elements, so their vectors of eight bytes are aligned too.  Elements of other rows, and those past the tensor's end, are left alone.
constexpr int RAGGED_BLOCKS = 7, RAGGED_COLUMNS = RAGGED_BLOCKS * MX_BLOCK;
struct Ragged {
  long long row, base;  // element that the warp's columns count from
  int block0, n;        // the row's block that the warp begins with; columns
  int c, first, next;   // this lane's first column (below 0: elements of what lies before), its first block (-1: those), and how many elements come before the next
  bool any;
  __device__ __forceinline__ Ragged(long long rows, int K, int groups) {
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), r = w / (uint32_t)groups;  // (32 bits: a division of 64 is as long as the rest of the kernel)
    row = r;
    block0 = (int)(w - r * (uint32_t)groups) * RAGGED_BLOCKS;
    base = row * K + block0 * MX_BLOCK;
    n = row < rows ? min(RAGGED_COLUMNS, K - block0 * MX_BLOCK) : 0;
    c = (int)(threadIdx.x & 31) * 8 - (int)(base & 7);
    any = c < n;
    first = c < 0 ? -1 : c / MX_BLOCK;
    next = (first + 1) * MX_BLOCK - c;
  }
  __device__ __forceinline__ bool in(int i) const { return c + i >= 0 && c + i < n; }
  __device__ __forceinline__ bool whole() const { return c >= 0 && c + 8 <= n; }
};
// All seven blocks, and 29 whole vectors inside the tensor: the elements before a boundary are the first ``phase`` of lanes 0, 4, ... 28, known to the compiler, so an
// element's block needs no comparison (8192 x 14343: 205 -> 113 us, and back 108 -> 97).
__device__ __forceinline__ bool seven(const Ragged& at, long long total) { return at.n == RAGGED_COLUMNS && at.base - (at.base & 7) + 8 * (4 * RAGGED_BLOCKS + 1) <= total; }
template <typename F>
__device__ __forceinline__ void with_phase(int phase, F f) {
  switch (phase) {
    case 0: return f(std::integral_constant<int, 0>{});
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    default: return f(std::integral_constant<int, 7>{});
  }
}
// bytes FROM ... TO - 1 of eight on an 8-byte boundary
template <int FROM, int TO>
__device__ __forceinline__ void put_bytes(uint8_t* to, const uint32_t (&w)[2]) {
  if constexpr (FROM < TO) {
    constexpr int SIZE = FROM % 4 == 0 && FROM + 4 <= TO ? 4 : FROM % 2 == 0 && FROM + 2 <= TO ? 2 : 1;
    const uint32_t v = w[FROM / 4] >> (8 * (FROM % 4));
    if (SIZE == 4) *reinterpret_cast<uint32_t*>(to + FROM) = v;
    else if (SIZE == 2) *reinterpret_cast<uint16_t*>(to + FROM) = (uint16_t)v;
    else to[FROM] = (uint8_t)v;
    put_bytes<FROM + SIZE, TO>(to, w);
  }
}
template <int PHASE, typename T>
__device__ __forceinline__ void quantize_seven(const T* x, uint8_t* codes, uint8_t* scales) {  // of the first lane's vector; of the first block
  const int lane = threadIdx.x & 31, last = PHASE ? 4 * RAGGED_BLOCKS : 4 * RAGGED_BLOCKS - 1;
  float f[8] = {};
  if (lane <= last) {
    Vec8<T> v;
    v.load(x + 8 * lane);
    v.to_float(f);
  }
  uint32_t lo = 0, hi = 0;  // largest magnitudes before and behind a boundary
#pragma unroll
  for (int i = 0; i < 8; ++i) (i < PHASE ? lo : hi) = max(i < PHASE ? lo : hi, __float_as_uint(f[i]) & 0x7fffffffu);
  const bool cut = (lane & 3) == 0;
  uint32_t top = cut ? hi : max(lo, hi);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (PHASE) top = max(top, __shfl_sync(0xffffffffu, lo, (lane | 3) + 1));  // (of the last four lanes nothing is kept)
  const uint32_t before = PHASE ? __shfl_up_sync(0xffffffffu, top, 1) : top, top_lo = cut && lane ? before : top;
  const uint32_t byte = mx_scale_byte<8>(top);
  const MxCoder<8> own(byte, top), first(mx_scale_byte<8>(top_lo), top_lo);
  if (lane > last) return;
  uint32_t w[2];
  auto word = [&](auto exact, int h) {
    constexpr bool E = decltype(exact)::value;
    auto one = [&](int i) { return (i < PHASE ? first : own).template add<E>(__float_as_uint(f[i])); };
    return MxCoder<8>::pack(one(4 * h), one(4 * h + 1), one(4 * h + 2), one(4 * h + 3));
  };
  if (own.exact && (PHASE == 0 || first.exact)) {
    w[0] = word(std::true_type{}, 0);
    w[1] = word(std::true_type{}, 1);
  } else {
    w[0] = word(std::false_type{}, 0);
    w[1] = word(std::false_type{}, 1);
  }
  uint8_t* to = codes + 8 * lane;
  if (PHASE && lane == 0) put_bytes<PHASE, 8>(to, w);
  else if (PHASE && lane == 4 * RAGGED_BLOCKS) put_bytes<0, PHASE>(to, w);
  else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  if (cut && lane < 4 * RAGGED_BLOCKS) scales[lane / 4] = (uint8_t)byte;
}
template <int PHASE, typename T>
__device__ __forceinline__ void dequantize_seven(const uint8_t* codes, const uint8_t* scales, T* y) {
  const int lane = threadIdx.x & 31, last = PHASE ? 4 * RAGGED_BLOCKS : 4 * RAGGED_BLOCKS - 1, block = lane / 4;
  if (lane > last) return;
  const uint2 w = *reinterpret_cast<const uint2*>(codes + 8 * lane);
  const bool cut = (lane & 3) == 0;
  const MxReader<8> own(block < RAGGED_BLOCKS ? scales[block] : MX_LOWEST<8>), first(PHASE && cut && lane ? scales[block - 1] : 0);
  float f[8], g[8];
  own.four(w.x, f);
  own.four(w.y, f + 4);
  if (PHASE && cut) {
    first.four(w.x, g);
    if (PHASE > 4) first.four(w.y, g + 4);
#pragma unroll
    for (int i = 0; i < PHASE; ++i) f[i] = g[i];
  }
  T* to = y + 8 * lane;
  if (PHASE && (lane == 0 || lane == 4 * RAGGED_BLOCKS)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i >= PHASE) == (lane == 0)) to[i] = T(f[i]);
  } else {
    Vec8<T> o;
    o.from_float(f);
    o.store(to);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_quantize_ragged_kernel(const T* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int blocks, int groups) {
  after_previous();
  const Ragged at(rows, K, groups);
  if (at.n == 0) return;  // (the whole warp)
  if (seven(at, rows * K)) {
    const int phase = (int)(at.base & 7);
    return with_phase(phase, [&](auto p) { quantize_seven<decltype(p)::value>(x + at.base - phase, codes + at.base - phase, scales + at.row * blocks + at.block0); });
  }
  float f[8] = {};
  if (at.any) {
    const long long e = at.base + at.c;
    if (e + 8 <= rows * K) {
      Vec8<T> v;
      v.load(x + e);
      v.to_float(f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = e + i < rows * K ? float(x[e + i]) : 0.f;
    }
  }
  if (!at.whole()) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = at.in(i) ? f[i] : 0.f;
  }
  uint32_t own = 0, after = 0;  // largest magnitudes of this lane's first block and of the one after
  if (at.next >= 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) own = max(own, __float_as_uint(f[i]) & 0x7fffffffu);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = __float_as_uint(f[i]) & 0x7fffffffu;
      if (i < at.next) own = max(own, m);
      else after = max(after, m);
    }
  }
  // Four lanes have the same first block, one after the other, counted from the lane that begins in block 0 or on it; the lane before them has the block's
  // first elements where it does not begin on a lane.
  const int lane = threadIdx.x & 31, from0 = (at.base & 7) != 0, l = lane - from0;
  const uint32_t before = __shfl_up_sync(0xffffffffu, after, 1);
  uint32_t top = lane > 0 && (l & 3) == 0 ? max(own, before) : own;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) top = max(top, __shfl_sync(0xffffffffu, top, (max(l, 0) ^ o) + from0));  // (lanes without columns may read any)
  const uint32_t top_after = __shfl_sync(0xffffffffu, top, l < 0 ? from0 : (l / 4 + 1) * 4 + from0);
  const uint32_t byte = mx_scale_byte<8>(top);
  if (l >= 0 && (l & 3) == 0 && at.first * MX_BLOCK < at.n) scales[at.row * blocks + at.block0 + at.first] = (uint8_t)byte;
  if (!at.any) return;
  const MxCoder<8> here(byte, top), there(mx_scale_byte<8>(top_after), top_after);
  uint32_t a[2];
  uint32_t u[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = __float_as_uint(f[k]);
  here.words(u, a);
  if (at.next < 8) {
    uint32_t b[2];
    there.words(u, b);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int own_bytes = max(0, min(4, at.next - 4 * h));
      const uint32_t mask = own_bytes == 4 ? 0xffffffffu : (1u << (8 * own_bytes)) - 1u;
      a[h] = (a[h] & mask) | (b[h] & ~mask);
    }
  }
  uint8_t* to = codes + at.base + at.c;
  if (at.whole()) {
    *reinterpret_cast<uint2*>(to) = make_uint2(a[0], a[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at.in(i)) to[i] = (uint8_t)(a[i / 4] >> (8 * (i % 4)));
  }
}
template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_ragged_kernel(const uint8_t* codes, const uint8_t* scales, T* y, long long rows, int K, int blocks,
                                                                   int groups) {
  after_previous();
  const Ragged at(rows, K, groups);
  if (seven(at, rows * K)) {
    const int phase = (int)(at.base & 7);
    return with_phase(phase, [&](auto p) { dequantize_seven<decltype(p)::value>(codes + at.base - phase, scales + at.row * blocks + at.block0, y + at.base - phase); });
  }
  if (!at.any) return;
  const long long e = at.base + at.c;
  uint2 w = make_uint2(0, 0);
  if (e + 8 <= rows * K) {
    w = *reinterpret_cast<const uint2*>(codes + e);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < rows * K) (i < 4 ? w.x : w.y) |= (uint32_t)codes[e + i] << (8 * (i % 4));
  }
  const uint8_t* s = scales + at.row * blocks + at.block0;
  const bool second = at.next < 8 && (at.first + 1) * MX_BLOCK < at.n;
  float f[8], g[8];
  const MxReader<8> here(at.first < 0 ? MX_LOWEST<8> : s[at.first]);
  here.four(w.x, f);
  here.four(w.y, f + 4);
  if (second) {
    const MxReader<8> there(s[at.first + 1]);
    there.four(w.x, g);
    there.four(w.y, g + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < at.next ? f[i] : g[i];
  }
  if (at.whole()) {
    Vec8<T> o;
    o.from_float(f);
    o.store(y + e);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at.in(i)) y[e + i] = T(f[i]);
  }
}

// The 16-bit codes of what gated_act_kernel takes, and back: a warp to a block, an element to a lane (only products in fp32 come here).
template <int BITS>
__device__ __forceinline__ uint32_t code(const MxCoder<BITS>& coder, uint32_t v) {
  const uint32_t pair[2] = {v, 0};
  uint32_t w[1];
  coder.words(pair, w);
  return w[0];
}
template <int BITS>
__global__ void __launch_bounds__(256) mx16_quantize_kernel(const float* x, uint16_t* codes, uint8_t* scales, uint32_t warps, int K, uint32_t blocks) {
  after_previous();
  const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), row = w / blocks, c = (w - row * blocks) * MX_BLOCK + (threadIdx.x & 31);
  if (w >= warps) return;
  const uint32_t v = c < (uint32_t)K ? __float_as_uint(x[(long long)row * K + c]) : 0u, top = __reduce_max_sync(0xffffffffu, v & 0x7fffffffu);
  const uint32_t byte = mx_scale_byte<BITS>(top);
  if (c < (uint32_t)K) codes[(long long)row * K + c] = (uint16_t)code(MxCoder<BITS>(byte, top), v);
  if ((threadIdx.x & 31) == 0) scales[w] = (uint8_t)byte;
}
template <int BITS>
__global__ void __launch_bounds__(256) mx16_dequantize_kernel(const uint16_t* codes, const uint8_t* scales, float* y, uint32_t warps, int K, uint32_t blocks) {
  after_previous();
  const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), row = w / blocks, c = (w - row * blocks) * MX_BLOCK + (threadIdx.x & 31);
  if (w >= warps || c >= (uint32_t)K) return;
  float f[2];
  MxReader<BITS>(scales[w]).two(codes[(long long)row * K + c], f);
  y[(long long)row * K + c] = f[0];
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

// x [R, K], codes [R, K], scales [R, ceil(K / 32)], all dense, x and codes on 16-byte bases.  Whole rows of blocks, rows of whole vectors, other rows:
// 8192 x 14336 bf16 53, 14344 75, 14343 113 us (and back 59, 68, 97).
template <typename T>
static int quantize(const T* x, uint8_t* codes, uint8_t* scales, long long R, long long K, cudaStream_t st) {
  const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK, groups = (blocks + RAGGED_BLOCKS - 1) / RAGGED_BLOCKS;
  if (K % MX_BLOCK == 0) return done(launch_after(mx8_quantize_kernel<T>, blocks_of(R * K / 16), 256, 0, st, x, codes, scales, R * K / 16));
  if (K % 8 == 0) return done(launch_after(mx8_quantize_vec_kernel<T>, blocks_of(R * blocks * 4), 256, 0, st, x, codes, scales, (uint32_t)R, (int)K, (uint32_t)blocks * 4));
  return done(launch_after(mx8_quantize_ragged_kernel<T>, blocks_of(R * groups * 32), 256, 0, st, x, codes, scales, R, (int)K, (int)blocks, (int)groups));
}
template <typename T>
static int dequantize(const uint8_t* codes, const uint8_t* scales, T* y, long long R, long long K, cudaStream_t st) {
  const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK, groups = (blocks + RAGGED_BLOCKS - 1) / RAGGED_BLOCKS;
  if (K % MX_BLOCK == 0) return done(launch_after(mx8_dequantize_kernel<T>, blocks_of(R * K / 16), 256, 0, st, codes, scales, y, R * K / 16));
  if (K % 8 == 0) return done(launch_after(mx8_dequantize_vec_kernel<T>, blocks_of(R * blocks * 4), 256, 0, st, codes, scales, y, (uint32_t)R, (int)K, (uint32_t)blocks * 4));
  return done(launch_after(mx8_dequantize_ragged_kernel<T>, blocks_of(R * groups * 32), 256, 0, st, codes, scales, y, R, (int)K, (int)blocks, (int)groups));
}
// (the threads of the forms for other rows are counted in 32 bits: 2^32 of them are 2^35 elements or, of a row of one element, 2^30)
static bool too_many(long long R, long long K) {
  const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
  return K > 0x7fffffe0ll || R > 0x7fffffffll * 64 / blocks || (K % MX_BLOCK && R > 0x3fffff00ll / blocks) || R * K / 16 / 256 >= 0x7fffffffll;
}
extern "C" int apb_mx8_quantize(const void* x, void* codes, void* scales, long long R, long long K, int is_bf16, cudaStream_t st) {
  if (R <= 0 || K <= 0) return 0;
  if (off16(x) || off16(codes) || too_many(R, K)) return 3;
  return is_bf16 ? quantize((const bf16*)x, (uint8_t*)codes, (uint8_t*)scales, R, K, st) : quantize((const float*)x, (uint8_t*)codes, (uint8_t*)scales, R, K, st);
}
extern "C" int apb_mx8_dequantize(const void* codes, const void* scales, void* y, long long R, long long K, int is_bf16, cudaStream_t st) {
  if (R <= 0 || K <= 0) return 0;
  if (off16(y) || off16(codes) || too_many(R, K)) return 3;
  return is_bf16 ? dequantize((const uint8_t*)codes, (const uint8_t*)scales, (bf16*)y, R, K, st)
                 : dequantize((const uint8_t*)codes, (const uint8_t*)scales, (float*)y, R, K, st);
}

// ``bits`` 16 or MX_HALF
extern "C" int apb_mx16_quantize(const float* x, void* codes, void* scales, long long R, int K, int bits, cudaStream_t st) {
  const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK, warps = R * blocks;
  if (warps <= 0) return 0;
  if (warps > 0xfffffff0ll || (bits != 16 && bits != MX_HALF)) return 3;
  return done(launch_after(bits == 16 ? mx16_quantize_kernel<16> : mx16_quantize_kernel<MX_HALF>, blocks_of(warps * 32), 256, 0, st, x, (uint16_t*)codes, (uint8_t*)scales, (uint32_t)warps, K, (uint32_t)blocks));
}
extern "C" int apb_mx16_dequantize(const void* codes, const void* scales, float* y, long long R, int K, int bits, cudaStream_t st) {
  const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK, warps = R * blocks;
  if (warps <= 0) return 0;
  if (warps > 0xfffffff0ll || (bits != 16 && bits != MX_HALF)) return 3;
  return done(launch_after(bits == 16 ? mx16_dequantize_kernel<16> : mx16_dequantize_kernel<MX_HALF>, blocks_of(warps * 32), 256, 0, st, (const uint16_t*)codes, (const uint8_t*)scales, y, (uint32_t)warps, K,
                           (uint32_t)blocks));
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
