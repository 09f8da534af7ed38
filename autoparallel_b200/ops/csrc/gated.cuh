// The middle of a gated feed-forward block: h = act(a) * b with a = x w1^T and b = x w3^T, and its derivative, as the ends of two products.
//
//   forward    both projections come out of one product, a and b of the same column of h in the same thread; h leaves in bf16, and for the backward
//              pass a and b, as codes of 8 or 16 bits (mx8.cuh).  Two forms of 16: fp16 numbers under the power of two of a block, off by 2^-11 of each value and
//              not by 2^-8 as bf16 would be, and whole numbers, off by 2^-15 of the block's largest value.  The gradients are off by 0.0024 of their size, not
//              0.0034 (both: da, db and the results are rounded to bf16); with whole numbers only while the values of a block are within some 150 times of each
//              other (a column 4096 times the others of its block: their weights' gradients off by 0.058 of their size).
//   backward   dh = dy w2 stays in fp32; da = dh b act'(a) and db = dh act(a) leave in bf16, and h, made again, for the gradient of w2
//
// ab, dab [M, 2, H]: a row of a (da), then the same row of b (db), so that one product makes the gradients of both weights.  The scales of codes are
// [M, 2, ceil(H / 32)].  H % 8 == 0.
#pragma once
#include <type_traits>

#include "mx8.cuh"
#include "ptx.cuh"

namespace apb {

enum : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

// Phi(-x) exp(x^2 / 2) for x >= 0, Phi the normal distribution: a polynomial in t = 1 / (1 + 0.275 x) without a constant, as the function falls off like
// 1 / x.  Fitted to the smallest largest relative error over all x (weighted least squares, the weights moved to where the error is): 2.2e-6.
__device__ __forceinline__ float normal_tail(float x) {
  const float t = __fdividef(1.f, fmaf(0.275f, x, 1.f));
  float p = -0.0552612767f;
  p = fmaf(p, t, 0.129859090f);
  p = fmaf(p, t, 0.00389011344f);
  p = fmaf(p, t, 0.103644602f);
  p = fmaf(p, t, 0.0981924608f);
  p = fmaf(p, t, 0.109972589f);
  p = fmaf(p, t, 0.109701321f);
  return p * t;
}

// act(a), and its derivative in ``d``, relative to the value: x / (1 + exp(-x)) keeps its digits where 1 + tanh would cancel, and a tail of the normal
// distribution those that 1 + erf would lose.  FINE: for fp32 results, by expf, erfcf and a true division, to a few units in the last place and what the rounding of
// an exponential's argument makes of it (the short forms: 2 + 1.2 |u| units for exp(u), some 70 of silu(-60)).  By the error function, 8192 x 4096 x 14336 backward: 988 us
// with erfc, 708 so (one of the sigmoids 708).
template <int ACT, bool FINE = false>
__device__ __forceinline__ float act_value(float a, float& d) {
  if (ACT == ACT_GELU) {
    const float e = FINE ? expf(-0.5f * a * a) : __expf(-0.5f * a * a);
    float phi;
    if (FINE) {
      phi = 0.5f * erfcf(-0.70710678f * a);
    } else {
      phi = e * normal_tail(fabsf(a));
      phi = a > 0.f ? 1.f - phi : phi;
    }
    d = fmaf(a * 0.39894228f, e, phi);
    return a * phi;
  }
  // silu: a s(a); gelu_tanh: a s(2 sqrt(2 / pi) (a + 0.044715 a^3)), s the logistic function
  float u = a, du = 1.f;
  if (ACT == ACT_GELU_TANH) {
    const float a2 = a * a;
    u = 1.59576912f * a * fmaf(0.044715f, a2, 1.f);
    du = fmaf(0.21406445f, a2, 1.59576912f);
  }
  const float s = FINE ? __fdiv_rn(1.f, 1.f + expf(-u)) : __fdividef(1.f, 1.f + __expf(-u));
  const float v = a * s;
  d = fmaf(v * (1.f - s), du, s);
  return v;
}

struct GatedOut {  // forward
  __nv_bfloat16* h;
  void* ab;  // codes
  uint8_t* scales;
  int act;
};
struct GatedGrad {  // backward
  const void* ab;  // codes
  const uint8_t* scales;
  __nv_bfloat16 *dab, *h;
  int act;
};

template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>{});
  else f(std::integral_constant<int, ACT_GELU_TANH>{});
}

// ---------------------------------------------------------------------------- a warp's 32 rows, 32 columns at a time, a row to a thread
// Staging in shared memory, 32 rows of 64 bytes: a thread writes or reads its own row, and the warp moves whole rows, four lanes to one.
__device__ __forceinline__ uint32_t stage64(int row, int unit) { return row * 64 + ((unit ^ (row >> 1 & 3)) << 4); }
__device__ __forceinline__ void stage_put(uint8_t* stg, int lane, const uint32_t (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stg + stage64(lane, i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
// rows row0 ... of ``dst`` (``ld`` elements apart), columns col ... col + 31 that are inside the matrix
__device__ __forceinline__ void stage_store(const uint8_t* stg, __nv_bfloat16* dst, long long ld, int row0, int col, int M, int H, int lane) {
  const int unit = lane & 3, sub = lane >> 2;
  if (col + unit * 8 >= H) return;
  __nv_bfloat16* p = dst + (long long)(row0 + sub) * ld + col + unit * 8;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = sub + 8 * j;
    if (row0 + row < M) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(stg + stage64(row, unit));
    p += 8 * ld;
  }
}
// the same for codes: rows of 32 bytes, in pieces of 8 (a row of b begins H bytes behind a's, which 8 divides)
__device__ __forceinline__ uint32_t stage32(int row, int unit) { return row * 32 + ((unit ^ (row >> 2 & 3)) << 3); }
__device__ __forceinline__ void stage_store8(const uint8_t* stg, uint8_t* dst, long long ld, int row0, int col, int M, int H, int lane) {
  const int unit = lane & 3, sub = lane >> 2;
  if (col + unit * 8 >= H) return;
  uint8_t* p = dst + (long long)(row0 + sub) * ld + col + unit * 8;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = sub + 8 * j;
    if (row0 + row < M) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(stg + stage32(row, unit));
    p += 8 * ld;
  }
}

// 32 values of a thread to codes in its row of the staging block; the scale byte
template <int BITS>
__device__ __forceinline__ uint32_t codes32(const uint32_t (&r)[32], uint8_t* stg, int lane) {
  const uint32_t top = mx_top(r), byte = mx_scale_byte<BITS>(top);
  const MxCoder<BITS> coder(byte, top);
  uint32_t w[8 * MX_BYTES<BITS>];
  coder.words(r, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BITS == 8) *reinterpret_cast<uint2*>(stg + stage32(lane, i)) = make_uint2(w[2 * i], w[2 * i + 1]);
    else *reinterpret_cast<uint4*>(stg + stage64(lane, i)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  return byte;
}

// Forward: columns col ... col + ncols - 1 of h from the accumulators at ``ta`` and ``tb``, and codes (BITS 0: none); ``stg``: 4096 bytes of the warp's own.
template <int BITS, typename Release>
__device__ __forceinline__ void gated_tile(const GatedOut& o, uint8_t* stg, uint32_t ta, uint32_t tb, int row0, int col, int ncols, int M, int H, int lane,
                                           Release release) {
  const int used = row0 < M ? min(ncols, H - col) : 0;  // (rows and columns past the matrix are not read)
  if (used <= 0) {
    release();
    return;
  }
  const int blocks = (H + MX_BLOCK - 1) / MX_BLOCK;
#pragma unroll 1
  for (int c = 0; c < used; c += 32) {
    uint32_t a[32], b[32], v[16];
    tmem_ld_32x32(ta + c, a);
    tmem_ld_32x32(tb + c, b);
    tmem_ld_wait_for(a);
    tmem_ld_wait_for(b);
    if (c + 32 >= used) release();
    with_act(o.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float d;
        const float h0 = act_value<decltype(act)::value>(__uint_as_float(a[2 * i]), d) * __uint_as_float(b[2 * i]);
        const float h1 = act_value<decltype(act)::value>(__uint_as_float(a[2 * i + 1]), d) * __uint_as_float(b[2 * i + 1]);
        v[i] = pack_bf16(h0, h1);
      }
    });
    __syncwarp();  // what was there before has been read
    stage_put(stg, lane, v);
    uint32_t sa = 0, sb = 0;
    if constexpr (BITS > 0) sa = codes32<BITS>(a, stg + 2048, lane);
    if constexpr (BITS == 8) sb = codes32<8>(b, stg + 2048 + 1024, lane);
    __syncwarp();
    stage_store(stg, o.h, H, row0, col + c, M, H, lane);
    if constexpr (BITS == 0) continue;
    if constexpr (BITS == 8) {
      uint8_t* codes = reinterpret_cast<uint8_t*>(o.ab);
      stage_store8(stg + 2048, codes, 2ll * H, row0, col + c, M, H, lane);
      stage_store8(stg + 2048 + 1024, codes + H, 2ll * H, row0, col + c, M, H, lane);
    } else if constexpr (BITS != 0) {
      __nv_bfloat16* codes = reinterpret_cast<__nv_bfloat16*>(o.ab);  // (two bytes each)
      stage_store(stg + 2048, codes, 2ll * H, row0, col + c, M, H, lane);
      __syncwarp();
      sb = codes32<BITS>(b, stg, lane);
      __syncwarp();
      stage_store(stg, codes + H, 2ll * H, row0, col + c, M, H, lane);
    }
    if (row0 + lane < M) {
      uint8_t* s = o.scales + (long long)(row0 + lane) * 2 * blocks + (col + c) / MX_BLOCK;
      s[0] = (uint8_t)sa;
      s[blocks] = (uint8_t)sb;
    }
  }
}

// The values a and b of a warp's 32 rows and 32 columns, on their way from memory to its staging block while the product is under way: whole rows, four
// lanes to one; rows and columns past the matrix are zeros.  16 bits: a's 32 x 64 bytes, then b's; 8 bits: 32 x 32 bytes each.
__device__ __forceinline__ void copy_async16(uint8_t* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async8(uint8_t* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 8 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int BITS>
struct AbFetch {
  uint32_t sa, sb;  // scale bytes of this thread's row
  __device__ __forceinline__ void start(const GatedGrad& g, uint8_t* stg, int row0, int col, int M, int H, int lane) {
    const int unit = lane & 3, sub = lane >> 2;
    const bool in = col + unit * 8 < H;
    const uint8_t* ab = reinterpret_cast<const uint8_t*>(g.ab);
    constexpr int SIZE = MX_BYTES<BITS>;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = sub + 8 * j;
      const bool ok = in && row0 + row < M;
      const uint8_t* src = ab + (ok ? (long long)(row0 + row) * 2 * H + col + unit * 8 : 0) * SIZE;  // (not read where it is not inside)
      const long long b = ok ? (long long)H * SIZE : 0;
      if (BITS == 8) {
        copy_async8(stg + stage32(row, unit), src, ok);
        copy_async8(stg + 1024 + stage32(row, unit), src + b, ok);
      } else {
        copy_async16(stg + stage64(row, unit), src, ok);
        copy_async16(stg + 2048 + stage64(row, unit), src + b, ok);
      }
    }
    sa = sb = MX_LOWEST<BITS>;
    if (row0 + lane < M && col < H) {
      const int blocks = (H + MX_BLOCK - 1) / MX_BLOCK;
      const uint8_t* s = g.scales + (long long)(row0 + lane) * 2 * blocks + col / MX_BLOCK;
      sa = s[0];
      sb = s[blocks];
    }
  }
};

// da, db and h of one element
template <int ACT, bool FINE = false>
__device__ __forceinline__ void gated_grad(float dh, float a, float b, float& da, float& db, float& h) {
  float d;
  const float v = act_value<ACT, FINE>(a, d);
  da = dh * b * d;
  db = dh * v;
  h = v * b;
}

// Backward: columns col ... of dh from the accumulator at ``taddr``.  ``fetch`` has started to bring the first 32 columns of a and b into ``stg``.
template <int BITS, typename Release>
__device__ __forceinline__ void gated_grad_tile(const GatedGrad& g, AbFetch<BITS>& fetch, uint8_t* stg, uint32_t taddr, int row0, int col, int ncols, int M,
                                                int H, int lane, Release release) {
  const int used = row0 < M ? min(ncols, H - col) : 0;
  copy_async_wait();
  if (used <= 0) {
    release();
    return;
  }
#pragma unroll 1
  for (int c = 0; c < used; c += 32) {
    uint32_t r[32], h[16];
    tmem_ld_32x32(taddr + c, r);
    copy_async_wait();
    __syncwarp();
    const MxReader<BITS> ra(fetch.sa), rb(fetch.sb);
    uint2 ca[BITS == 8 ? 4 : 1], cb[BITS == 8 ? 4 : 1];
    if constexpr (BITS == 8) {  // (this thread's codes, before da and db take their place)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ca[i] = *reinterpret_cast<const uint2*>(stg + stage32(lane, i));
        cb[i] = *reinterpret_cast<const uint2*>(stg + 1024 + stage32(lane, i));
      }
      __syncwarp();
    }
    tmem_ld_wait_for(r);
    if (c + 32 >= used) release();
    with_act(g.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // eight columns at a time, in this thread's row: a and b out, da and db into their place
        uint4* pa = reinterpret_cast<uint4*>(stg + stage64(lane, i));
        uint4* pb = reinterpret_cast<uint4*>(stg + 2048 + stage64(lane, i));
        float a[8], b[8];
        if constexpr (BITS == 8) {
          ra.four(ca[i].x, a);
          ra.four(ca[i].y, a + 4);
          rb.four(cb[i].x, b);
          rb.four(cb[i].y, b + 4);
        } else {
          const uint4 x = *pa, y = *pb;
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            ra.two(xs[k], a + 2 * k);
            rb.two(ys[k], b + 2 * k);
          }
        }
        float da[8], db[8], v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) gated_grad<decltype(act)::value>(__uint_as_float(r[8 * i + k]), a[k], b[k], da[k], db[k], v[k]);
        *pa = make_uint4(pack_bf16(da[0], da[1]), pack_bf16(da[2], da[3]), pack_bf16(da[4], da[5]), pack_bf16(da[6], da[7]));
        *pb = make_uint4(pack_bf16(db[0], db[1]), pack_bf16(db[2], db[3]), pack_bf16(db[4], db[5]), pack_bf16(db[6], db[7]));
#pragma unroll
        for (int k = 0; k < 4; ++k) h[4 * i + k] = pack_bf16(v[2 * k], v[2 * k + 1]);
      }
    });
    __syncwarp();
    stage_store(stg, g.dab, 2ll * H, row0, col + c, M, H, lane);
    stage_store(stg + 2048, g.dab + H, 2ll * H, row0, col + c, M, H, lane);
    __syncwarp();
    stage_put(stg, lane, h);
    __syncwarp();
    stage_store(stg, g.h, H, row0, col + c, M, H, lane);
    __syncwarp();
    if (c + 32 < used) fetch.start(g, stg, row0, col + c + 32, M, H, lane);
  }
}

// ---------------------------------------------------------------------------- four columns of a row to a thread, eight threads to 32 columns
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) { return make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); }
// The eight threads come together, those with columns past the matrix (whose a and b are zeros) among them.  8 bits: the codes in .x.
template <int BITS>
__device__ __forceinline__ uint2 codes4(const float (&v)[4], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const uint32_t eight = 0xffu << (threadIdx.x & 24);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(eight, top, o));
  byte = mx_scale_byte<BITS>(top);
  const MxCoder<BITS> coder(byte, top);
  const uint32_t u[4] = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  uint32_t w[MX_BYTES<BITS>];
  coder.words(u, w);
  return make_uint2(w[0], BITS == 8 ? 0 : w[MX_BYTES<BITS> - 1]);
}
template <int BITS>
__device__ __forceinline__ void gated_four(const GatedOut& o, long long row, int col, int H, const float (&a)[4], const float (&b)[4]) {
  float h[4];
  with_act(o.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float d;
      h[i] = act_value<decltype(act)::value>(a[i], d) * b[i];
    }
  });
  const bool in = col < H;
  if (in) *reinterpret_cast<uint2*>(o.h + row * H + col) = pack4(h);
  if constexpr (BITS == 0) return;
  uint32_t sa = 0, sb = 0;
  const long long at = row * 2 * H + col;
  if constexpr (BITS == 8) {
    const uint2 ca = codes4<8>(a, sa), cb = codes4<8>(b, sb);
    if (!in) return;
    uint8_t* codes = reinterpret_cast<uint8_t*>(o.ab) + at;
    *reinterpret_cast<uint32_t*>(codes) = ca.x;
    *reinterpret_cast<uint32_t*>(codes + H) = cb.x;
  } else if constexpr (BITS != 0) {
    const uint2 ca = codes4<BITS>(a, sa), cb = codes4<BITS>(b, sb);
    if (!in) return;
    uint16_t* codes = reinterpret_cast<uint16_t*>(o.ab) + at;
    *reinterpret_cast<uint2*>(codes) = ca;
    *reinterpret_cast<uint2*>(codes + H) = cb;
  }
  if (col % MX_BLOCK == 0) {
    const int blocks = (H + MX_BLOCK - 1) / MX_BLOCK;
    uint8_t* s = o.scales + row * 2 * blocks + col / MX_BLOCK;
    s[0] = (uint8_t)sa;
    s[blocks] = (uint8_t)sb;
  }
}
// a and b of four columns as they lie in memory (8 bits: .x), and the scale bytes
template <int BITS>
struct AbFour {
  uint2 a, b;
  uint32_t sa, sb;
  __device__ __forceinline__ void load(const GatedGrad& g, long long row, int col, int H) {
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(g.ab) + (row * 2 * H + col) * MX_BYTES<BITS>;
    if (BITS == 8) {
      a.x = *reinterpret_cast<const uint32_t*>(codes);
      b.x = *reinterpret_cast<const uint32_t*>(codes + H);
    } else {
      a = *reinterpret_cast<const uint2*>(codes);
      b = *reinterpret_cast<const uint2*>(codes + 2ll * H);
    }
    const int blocks = (H + MX_BLOCK - 1) / MX_BLOCK;
    const uint8_t* s = g.scales + row * 2 * blocks + col / MX_BLOCK;
    sa = s[0];
    sb = s[blocks];
  }
};
template <int BITS>
__device__ __forceinline__ void gated_grad_four(const GatedGrad& g, const AbFour<BITS>& ab, long long row, int col, int H, const float (&dh)[4]) {
  float a[4], b[4], da[4], db[4], h[4];
  const long long at = row * 2 * H + col;
  const MxReader<BITS> ra(ab.sa), rb(ab.sb);
  if constexpr (BITS == 8) {
    ra.four(ab.a.x, a);
    rb.four(ab.b.x, b);
  } else {
    ra.two(ab.a.x, a);
    ra.two(ab.a.y, a + 2);
    rb.two(ab.b.x, b);
    rb.two(ab.b.y, b + 2);
  }
  with_act(g.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 4; ++i) gated_grad<decltype(act)::value>(dh[i], a[i], b[i], da[i], db[i], h[i]);
  });
  *reinterpret_cast<uint2*>(g.dab + at) = pack4(da);
  *reinterpret_cast<uint2*>(g.dab + at + H) = pack4(db);
  *reinterpret_cast<uint2*>(g.h + row * H + col) = pack4(h);
}

}  // namespace apb
