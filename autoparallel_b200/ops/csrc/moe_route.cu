// Routing of tokens to experts: scores, choice of the top k (of the top groups), gate weights, and the gradient of the logits.
// Semantics in ops/moe_ops.py; everything in fp32, in one pass over the logits.
//
// L lanes have a token, V experts each, all in registers; the k best are found by k rounds of "largest, lowest index first".  That takes instructions, and
// they are the bound, not memory (131072 x 128: 69 % of the issue slots, 13 % of DRAM; backward 52 and 26), so a token has the fewest lanes that hold it.
//   forward   8192 x 64 bf16, 8 of softmax: 2.6 us, 131072 x 64: 16.3, 131072 x 128, 6, with bias: 27.2 (1.5 TB/s); 16383 x 256 fp32 sigmoid, 8 of the 4 best
//             of 8 groups, with bias: 21.6, 65536 x 256 bf16 the same way: 50.6, without groups 41.8, without bias 29.5, of softmax 25.0
//   backward  2.1, 7.9, 15.6 (4.5 TB/s), 8.0, 13.7, 13.8: the scores are computed again from the logits, which the forward would write as 4 bytes an expert
//             for this to read; a choice's gradient is written by the lane that has the choice, so there are no atomics
//
// This file is compiled without --use_fast_math: the choice between two experts hangs on the last bit of a sigmoid, and has to be the same
// wherever the formula is evaluated as written (expf, IEEE division, denormals kept).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <type_traits>

#include "launch.cuh"

namespace apb {

constexpr int ROUTE_WARPS = 8, ROUTE_MAX_GROUPS = 64;

struct RouteParams {
  const void* x;
  const float* bias;
  float* w;
  long long* idx;
  long long tokens;
  int E, k, groups, size, top_groups, renorm, vec;
  float scale;
  uint32_t mask;  // 2^b - 1, at least E - 1
};

template <typename T>
__device__ __forceinline__ float route_load(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *p;
  else return __bfloat162float(*p);
}
// V elements of a row from ``e0`` on; those past E are -inf
template <typename T, int V>
__device__ __forceinline__ void route_load_row(const T* row, int e0, int E, bool vec, float (&x)[V]) {
  if (vec) {
    constexpr int PER = 16 / sizeof(T);
    uint4 v[V / PER];
#pragma unroll
    for (int c = 0; c < V / PER; ++c) {
      constexpr uint32_t NONE = std::is_same<T, float>::value ? 0xFF800000u : 0xFF80FF80u;
      v[c] = make_uint4(NONE, NONE, NONE, NONE);
      if (e0 + c * PER < E) v[c] = *reinterpret_cast<const uint4*>(row + e0 + c * PER);
    }
#pragma unroll
    for (int c = 0; c < V / PER; ++c) {
      const uint32_t u[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          x[c * PER + i] = __uint_as_float(u[i]);
        } else {
          x[c * PER + 2 * i] = __uint_as_float(u[i] << 16);
          x[c * PER + 2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = e0 + i < E ? route_load(row + e0 + i) : -CUDART_INF_F;
  }
}

__device__ __forceinline__ float route_sigmoid(float x) { return __frcp_rn(1.0f + expf(-x)); }
// e^x and the sigmoid from the hardware's approximations: e^x to a few 1e-7 of itself for |x| up to 10 or so, the sigmoid to 5e-7 absolute
// (the error of e^-x grows with |x|, its weight in the sigmoid falls faster).
__device__ __forceinline__ float route_exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ float route_sigmoid_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + route_exp_fast(-x)));
  return y;
}

// Order of the floats as unsigned integers.  -0 counts as 0 and every NaN as the same one, larger than all numbers: the sum with 0 makes
// them so (the result of an addition is the canonical NaN).  0 is smaller than the order of any float.
__device__ __forceinline__ uint32_t route_order(float c) {
  const uint32_t u = __float_as_uint(c + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_unorder(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < L; d *= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int d = 1; d < L; d *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int d = 1; d < L; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// How far two choice values have to be apart for their order to be sure, when they come from the fast sigmoid: twice its error, and the rounding of
// the sum with the bias.
__device__ __forceinline__ float route_margin(float c) { return 1e-6f + 2.4e-7f * fabsf(c); }

// Whether all experts with keys in the range of ``key`` have the logit ``x``: the sigmoids of its neighbours among the bf16 numbers lie outside.  (Among the
// fp32 numbers they never do.  Neighbours of 0 and of infinities come out as NaN or too close: no.)
template <typename T>
__device__ __forceinline__ bool route_alone(float x, uint32_t key, uint32_t mask) {
  if (std::is_same<T, float>::value) return false;
  const uint32_t u = __float_as_uint(x);
  const float a = route_sigmoid_fast(__uint_as_float(u + 0x10000u)), b = route_sigmoid_fast(__uint_as_float(u - 0x10000u)), m = 2.f * route_margin(1.f);
  return fmaxf(a, b) - route_unorder(key | mask) > m && route_unorder(key & ~mask) - fminf(a, b) > m;
}

// Orders of the choice values of a lane's experts; 0 for what cannot be chosen.
template <typename T, int V, bool SIGMOID, bool FAST>
__device__ __forceinline__ void route_values(const RouteParams& p, int e0, const float (&x)[V], uint32_t (&o)[V]) {
  float c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = !SIGMOID ? x[i] : FAST ? route_sigmoid_fast(x[i]) : route_sigmoid(x[i]);
  if (p.bias != nullptr) {
    if (p.vec) {  // (a multiple of 4 experts: in or out together)
#pragma unroll
      for (int i = 0; i < V; i += 4)
        if (e0 + i < p.E) {
          const float4 b = *reinterpret_cast<const float4*>(p.bias + e0 + i);
          c[i] += b.x, c[i + 1] += b.y, c[i + 2] += b.z, c[i + 3] += b.w;
        }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e0 + i < p.E) c[i] += p.bias[e0 + i];
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = e0 + i < p.E ? route_order(c[i]) : 0u;
}

// The experts outside a token's best groups get order 0.  Returns whether the fast values leave the choice of groups open.
//
// Groups of whole lanes (32 of 256 experts on 16 lanes of 16) stay in registers; others go through shared memory, a lane a group.
template <int L, int V>
constexpr int route_row_words() { return L * V + L * V / 32 + 1; }  // (one word more every 32: groups of 32 begin in different banks)
template <int L, int V>
constexpr int route_smem() { return ROUTE_WARPS * (32 / L) * (route_row_words<L, V>() + ROUTE_MAX_GROUPS) * 4; }
template <int L, int V, bool SIGMOID, bool FAST>
__device__ __forceinline__ bool route_groups(const RouteParams& p, int warp, int tok, int sub, uint32_t (&o)[V]) {
  extern __shared__ uint32_t route_words[];
  auto value = [&](uint32_t a, uint32_t b) { return SIGMOID && p.size > 1 ? route_order(route_unorder(a) + route_unorder(b)) : a; };
  // A sum of unlike signs is smaller than what was rounded for it, which the margin below does not count: up to 1 it is within what the margin has to
  // spare (the two sigmoids differ by 1.8e-7 at most, of 5e-7), beyond that nothing is sure.
  auto cancels = [&](uint32_t a, uint32_t b) { return SIGMOID && FAST && p.size > 1 && route_unorder(a) > 1.f && route_unorder(b) < -1.f; };
  bool vague = false;
  uint32_t kept_min = 0xFFFFFFFFu, dropped_max = 0;
  if (p.size % V == 0) {
    const int per = p.size / V, g = sub / per, first = g * per;
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (SIGMOID) b = max(b, min(a, o[i]));
      a = max(a, o[i]);
    }
    const uint32_t a0 = a, b0 = b;
    for (int d = 1; d < per; ++d) {
      const int from = tok * L + first + (sub - first + d) % per;
      const uint32_t a1 = __shfl_sync(0xffffffffu, a0, from & 31), b1 = __shfl_sync(0xffffffffu, b0, from & 31);
      b = max(max(b, b1), min(a, a1));
      a = max(a, a1);
    }
    const uint32_t mine = g < p.groups ? value(a, b) : 0u;
    vague = cancels(a, b);
    int before = 0;
    for (int h = 0; h < p.groups; ++h) {
      const uint32_t v = __shfl_sync(0xffffffffu, mine, tok * L + h * per);
      before += v > mine || (v == mine && h < g);
    }
    const bool kept = before < p.top_groups;
    if (kept) kept_min = mine;
    else dropped_max = mine;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = kept ? o[i] : 0u;
  } else {
    constexpr int WORDS = route_row_words<L, V>() + ROUTE_MAX_GROUPS;
    uint32_t *row = route_words + (warp * (32 / L) + tok) * WORDS, *val = row + route_row_words<L, V>();
#pragma unroll
    for (int i = 0; i < V; ++i) row[sub * V + i + (sub * V + i) / 32] = o[i];
    __syncwarp();
    for (int g = sub; g < p.groups; g += L) {
      uint32_t a = 0, b = 0;
      for (int i = 0; i < p.size; ++i) {
        const int e = g * p.size + i;
        const uint32_t v = row[e + e / 32];
        b = max(b, min(a, v));
        a = max(a, v);
      }
      val[g] = value(a, b);
      vague |= cancels(a, b);
    }
    __syncwarp();
    unsigned long long kept = 0;  // bit i: this lane's i-th group
    for (int g = sub, i = 0; g < p.groups; g += L, ++i) {
      const uint32_t mine = val[g];
      int before = 0;
      for (int h = 0; h < p.groups; ++h) before += val[h] > mine || (val[h] == mine && h < g);
      if (before < p.top_groups) {
        kept |= 1ull << i;
        kept_min = min(kept_min, mine);
      } else {
        dropped_max = max(dropped_max, mine);
      }
    }
    __syncwarp();
    for (int g = sub, i = 0; g < p.groups; g += L, ++i) val[g] = kept >> i & 1;
    __syncwarp();
    int g = sub * V / p.size, r = sub * V - g * p.size;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (g < p.groups && !val[g]) o[i] = 0;
      if (++r == p.size) {
        r = 0;
        ++g;
      }
    }
    __syncwarp();
  }
  if (!SIGMOID || !FAST) return false;
  const uint32_t lowest = ~lanes_max<L>(~kept_min), highest = lanes_max<L>(dropped_max);
  if (highest == 0) return false;
  const float low = route_unorder(lowest);
  return vague || !(low - route_unorder(highest) > 2.f * route_margin(low));
}

// Lane j's choice from whole values and numbers: the largest (value, -number) below the last.
template <int L, int V>
__device__ __forceinline__ int route_select_exact(const uint32_t (&o)[V], int e0, int k, int sub) {
  uint32_t lo = 0xFFFFFFFFu;
  int le = -1, mine = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t bo = 0;
    int be = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if ((o[i] < lo || (o[i] == lo && e0 + i > le)) && o[i] > bo) {
        bo = o[i];
        be = e0 + i;
      }
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
      const uint32_t ho = __shfl_xor_sync(0xffffffffu, bo, d);
      const int he = __shfl_xor_sync(0xffffffffu, be, d);
      if (ho > bo || (ho == bo && he < be)) {
        bo = ho;
        be = he;
      }
    }
    lo = bo;
    le = be;
    if (sub == j) mine = be;
  }
  return mine;
}

// L lanes hold a token, V experts each (lane after lane), and lane j ends up with its j-th choice: k <= L.
//
// The choice takes keys in place of the choice values: the upper bits of the value's order, and in the lower b bits (2^b >= E) the expert's number,
// inverted, so that the larger of two keys is the one to be chosen.  All keys differ, which makes a step of the selection - the largest key below
// the last - max(key - last) + last in wrapping arithmetic: two instructions a key.  Two things are left out at first: the lower bits of a
// value, and for sigmoid scores the last bits of a sigmoid, which is taken from the hardware's approximations (softmax of bf16 logits without bias: neither,
// the keys have all their 16 bits).  So the choice is proved afterwards.  Its own experts have to stand in the order of their exact values, neighbour by
// neighbour.  And the rest has to lie below the last of them.  Where the range of values that the rest's largest key stands for comes close (1 token in
// 100, or 1 in 5 for equal bf16 logits), that expert's exact value is compared, and one more step of the selection gives the range of all the
// others: a key names the lowest number of its range, not the largest value.  Others in the same range do no harm if they can only have the same logit.
// Where the proof fails, the warp does the choice again with exact values and numbers.
//
// (48, 64 and 80 registers for 8, 16 and 32 experts a lane: left to itself the compiler takes a few more for the code that few warps come to.)
template <typename T, int L, int V, bool SIGMOID>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, V == 8 ? 5 : V == 16 ? 4 : 3) moe_route_kernel(RouteParams p) {
  after_previous();
  constexpr int TPW = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tok = lane / L, sub = lane % L;
  const long long t = ((long long)blockIdx.x * ROUTE_WARPS + warp) * TPW + tok;
  const bool in = t < p.tokens;
  const T* row = reinterpret_cast<const T*>(p.x) + (in ? t : p.tokens - 1) * p.E;  // (lanes without a token follow the last one)
  const int e0 = sub * V;
  const bool chosen = sub < p.k;
  float m_all = -CUDART_INF_F, total_all = 0.f;
  const bool proved = SIGMOID || std::is_same<T, float>::value || p.bias != nullptr;
  auto range = [&](uint32_t key) { return key & ~p.mask; };
  uint32_t mine = 0, last = 0, others = 0;  // keys: this lane's choice, the largest of the rest, the one after it (0: there is none)
  bool unsure, near = false;                // near: the last choice to the range of the rest's largest key
  {
    float x[V];
    uint32_t o[V], key[V];
    route_load_row<T, V>(row, e0, p.E, p.vec, x);
    if (!SIGMOID && !p.renorm) {
#pragma unroll
      for (int i = 0; i < V; ++i) m_all = fmaxf(m_all, x[i]);
      m_all = lanes_max<L>(m_all);
      if (m_all == -CUDART_INF_F) m_all = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) total_all += route_exp_fast(x[i] - m_all);
      total_all = lanes_sum<L>(total_all);
    }
    route_values<T, V, SIGMOID, true>(p, e0, x, o);
    unsure = p.groups > 1 && route_groups<L, V, SIGMOID, true>(p, warp, tok, sub, o);
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = o[i] == 0 ? 0u : (o[i] & ~p.mask) | (p.mask - (e0 + i));
#pragma unroll
    for (int i = 0; i < V; ++i) last = max(last, key[i]);
    last = lanes_max<L>(last);
    for (int j = 0; j < p.k; ++j) {
      if (sub == j) mine = last;
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) best = max(best, key[i] - last);
      last += lanes_max<L>(best);
    }
    if (proved) {
      near = sub + 1 == p.k && last != 0;
      if (SIGMOID) {
        const float lo = route_unorder(range(mine));
        near = near && !(lo - route_unorder(last | p.mask) > route_margin(lo));
      } else {
        near = near && range(mine) == range(last) && range(last) != range(0x007FFFFFu);  // (-inf has a range to itself)
      }
      if (__any_sync(0xffffffffu, near)) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) best = max(best, key[i] - last);
        others = last + lanes_max<L>(best);
      }
    }
  }
  int e = mine != 0 ? (int)(p.mask - (mine & p.mask)) : 0;
  float xe = route_load(row + e), se = SIGMOID ? route_sigmoid(xe) : 0.f;
  if (proved) {
    auto before = [](float c0, int e0, float c1, int e1) { return c0 > c1 || (c0 == c1 && e0 < e1); };
    auto value = [&](float x, float s, int i) { return (SIGMOID ? s : x) + (p.bias != nullptr ? p.bias[i] : 0.f); };
    const float c = value(xe, se, e), next_c = __shfl_down_sync(0xffffffffu, c, 1, L);
    const int next_e = __shfl_down_sync(0xffffffffu, e, 1, L);
    unsure |= sub + 1 < p.k && !before(c, e, next_c, next_e);
    if (near) {
      const int r = (int)(p.mask - (last & p.mask));
      const float xr = route_load(row + r);
      const bool tie = p.bias == nullptr && xr == xe;  // (the keys have them in the order of their numbers)
      bool open = others != 0 && (SIGMOID ? !(c - route_unorder(others | p.mask) > route_margin(c)) : range(others) == range(last));
      if (SIGMOID && open && tie) open = !route_alone<T>(xe, last, p.mask);
      unsure |= open || !(tie || before(c, e, value(xr, SIGMOID ? route_sigmoid(xr) : 0.f, r), r));
    }
    if (__any_sync(0xffffffffu, unsure)) {
      float x[V];
      uint32_t o[V];
      route_load_row<T, V>(row, e0, p.E, p.vec, x);
      route_values<T, V, SIGMOID, false>(p, e0, x, o);
      if (p.groups > 1) route_groups<L, V, SIGMOID, false>(p, warp, tok, sub, o);
      e = route_select_exact<L, V>(o, e0, p.k, sub);
      xe = route_load(row + e);
      se = SIGMOID ? route_sigmoid(xe) : 0.f;
    }
  }
  float s, total;
  if (SIGMOID) {
    s = chosen ? se : 0.f;
    total = p.renorm ? lanes_sum<L>(s) : 1.f;
  } else if (p.renorm) {
    float m = lanes_max<L>(chosen ? xe : -CUDART_INF_F);
    if (m == -CUDART_INF_F) m = 0.f;
    s = chosen ? expf(xe - m) : 0.f;
    total = lanes_sum<L>(s);
  } else {
    s = expf(xe - m_all);
    total = total_all;
  }
  if (in && chosen) {
    p.w[t * p.k + sub] = (total == 0.f ? 0.f : s / total) * p.scale;
    p.idx[t * p.k + sub] = e;
  }
}

struct RouteBwdParams {
  const float* dw;
  const void* x;
  const long long* idx;
  void* dx;
  long long tokens;
  int E, k, renorm, vec;
  float scale;
};

template <typename T, int V>
__device__ __forceinline__ void route_store_row(T* row, int e0, int E, bool vec, const float (&v)[V]) {
  if (vec) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < V / PER; ++c) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          u[i] = __float_as_uint(v[c * PER + i]);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[c * PER + 2 * i], v[c * PER + 2 * i + 1]);
          u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      if (e0 + c * PER < E) *reinterpret_cast<uint4*>(row + e0 + c * PER) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e0 + i < E) {
        if constexpr (std::is_same<T, float>::value) row[e0 + i] = v[i];
        else row[e0 + i] = __float2bfloat16(v[i]);
      }
  }
}

// With p the weights before the scale and g = dweights * scale:
//   softmax over the chosen  dx_j = p_j (g_j - sum g p)          softmax over all  dx_e = p_e (g_e - sum g p), g_e = 0 for the others
//   sigmoid                  dx_j = g_j s_j (1 - s_j), with the sum of the chosen S: g_j <- (g_j - sum g p) / S first
// The row is written whole (zeros, or the gradient of the experts that were not chosen), then the chosen ones over it.
template <typename T, int L, int V, bool SIGMOID>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) moe_route_bwd_kernel(RouteBwdParams p) {
  after_previous();
  constexpr int TPW = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tok = lane / L, sub = lane % L;
  const long long t = ((long long)blockIdx.x * ROUTE_WARPS + warp) * TPW + tok;
  const bool in = t < p.tokens;
  const long long tt = in ? t : p.tokens - 1;
  const T* row = reinterpret_cast<const T*>(p.x) + tt * p.E;
  T* out = reinterpret_cast<T*>(p.dx) + tt * p.E;
  const int e0 = sub * V;
  long long e = sub < p.k ? p.idx[tt * p.k + sub] : -1;
  const bool chosen = e >= 0 && e < p.E;  // (a number that names no expert has no gradient)
  const float g = chosen ? p.dw[tt * p.k + sub] * p.scale : 0.f;
  const float xe = chosen ? route_load(row + e) : -CUDART_INF_F;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  float mine;
  if (SIGMOID) {
    const float s = chosen ? route_sigmoid(xe) : 0.f;
    float ds = g;
    if (p.renorm) {
      const float total = lanes_sum<L>(s), q = total == 0.f ? 0.f : s / total;  // (1 for a single choice: no gradient, not a rounding error's)
      const float dot = lanes_sum<L>(g * q);  // (by every lane: tokens whose scores are all zero share warps with others)
      ds = total == 0.f ? 0.f : (g - dot) / total;
    }
    mine = ds * s * (chosen ? route_sigmoid(-xe) : 0.f);  // (1 - s, also where s rounds to 1)
  } else if (p.renorm) {
    float m = lanes_max<L>(xe);
    if (m == -CUDART_INF_F) m = 0.f;
    const float s = chosen ? expf(xe - m) : 0.f, total = lanes_sum<L>(s), q = total == 0.f ? 0.f : s / total;
    mine = q * (g - lanes_sum<L>(g * q));
  } else {
    float x[V];
    route_load_row<T, V>(row, e0, p.E, p.vec, x);
    float m = -CUDART_INF_F, total = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
    m = lanes_max<L>(m);
    if (m == -CUDART_INF_F) m = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = route_exp_fast(x[i] - m);
      total += x[i];
    }
    total = lanes_sum<L>(total);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const float q = chosen ? expf(xe - m) * inv : 0.f, dot = lanes_sum<L>(g * q);
    mine = q * (g - dot);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = x[i] * inv * -dot;
  }
  if (in) route_store_row<T, V>(out, e0, p.E, p.vec, v);
  __syncwarp();
  if (in && chosen) {
    if constexpr (std::is_same<T, float>::value) out[e] = mine;
    else out[e] = __float2bfloat16(mine);
  }
}

// f(L, V) for the smallest number of lanes that holds the experts, up to 16 a lane, and a choice a lane.  Forward, us, this / twice the lanes / twice the
// experts a lane: 131072 x 64 16.7 / 33.3 / 24.3, 131072 x 128 27.4 / 35.6, 65536 x 256 in groups 53.5 / 67.1 / 66.9, without 25.6 / 34.8 / 21.7 (32 experts a
// lane would be faster there alone).
template <typename F>
static int route_shape(int E, int k, F f) {
  auto c = [](auto v) { return v; };
#define APB_ROUTE(L, V) return f(c(std::integral_constant<int, L>{}), c(std::integral_constant<int, V>{}))
  if (k <= 4 && E <= 32) APB_ROUTE(4, 8);
  if (k <= 8 && E <= 64) APB_ROUTE(8, 8);
  if (k <= 8 && E <= 128) APB_ROUTE(8, 16);
  if (k <= 16 && E <= 128) APB_ROUTE(16, 8);
  if (k <= 16 && E <= 256) APB_ROUTE(16, 16);
  if (E <= 256) APB_ROUTE(32, 8);
  if (E <= 512) APB_ROUTE(32, 16);
  APB_ROUTE(32, 32);
#undef APB_ROUTE
}
static bool route_args_ok(long long tokens, int E, int k) { return tokens >= 0 && E >= 1 && E <= 1024 && k >= 1 && k <= 32 && k <= E; }
template <int L>
static dim3 route_grid(long long tokens) {
  constexpr int PER = ROUTE_WARPS * (32 / L);
  return dim3((unsigned)((tokens + PER - 1) / PER));
}

}  // namespace apb

using namespace apb;

// logits [tokens, E] (bf16 or fp32, rows after each other, 16-byte base), bias fp32 [E] (16-byte base) or null -> w fp32 [tokens, k], idx [tokens, k].
// Returns 0, or an argument / launch error (nothing launched).
extern "C" int apb_moe_route(const void* logits, const float* bias, float* w, long long* idx, long long tokens, int E, int k, int sigmoid, int groups,
                             int top_groups, int renorm, float scale, int is_bf16, cudaStream_t st) {
  if (!route_args_ok(tokens, E, k) || groups < 1 || groups > ROUTE_MAX_GROUPS || E % groups || top_groups < 1 || top_groups > groups ||
      k > top_groups * (E / groups) || ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(bias)) & 15))
    return 3;
  if (tokens == 0) return 0;
  uint32_t mask = 1;
  while ((int)mask < E - 1) mask = 2 * mask + 1;
  const RouteParams p{logits, bias, w, idx, tokens, E, k, groups, E / groups, top_groups, renorm, E % (is_bf16 ? 8 : 4) == 0, scale, mask};
  return route_shape(E, k, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    const size_t smem = groups > 1 && p.size % V != 0 ? route_smem<L, V>() : 0;
    static_assert(route_smem<L, V>() <= 48 * 1024, "shared memory without opting in");
    auto launch = [&](auto kern) { launch_after(kern, route_grid<L>(tokens), 32 * ROUTE_WARPS, smem, st, p); };
    if (is_bf16) sigmoid ? launch(moe_route_kernel<__nv_bfloat16, L, V, true>) : launch(moe_route_kernel<__nv_bfloat16, L, V, false>);
    else sigmoid ? launch(moe_route_kernel<float, L, V, true>) : launch(moe_route_kernel<float, L, V, false>);
    return cudaGetLastError() == cudaSuccess ? 0 : 4;
  });
}

// dw fp32 [tokens, k], logits and dx [tokens, E], idx [tokens, k].
extern "C" int apb_moe_route_bwd(const float* dw, const void* logits, const long long* idx, void* dx, long long tokens, int E, int k, int sigmoid,
                                 int renorm, float scale, int is_bf16, cudaStream_t st) {
  if (!route_args_ok(tokens, E, k) || ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dx)) & 15)) return 3;
  if (tokens == 0) return 0;
  const RouteBwdParams p{dw, logits, idx, dx, tokens, E, k, renorm, E % (is_bf16 ? 8 : 4) == 0, scale};
  return route_shape(E, k, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    auto launch = [&](auto kern) { launch_after(kern, route_grid<L>(tokens), 32 * ROUTE_WARPS, 0, st, p); };
    if (is_bf16) sigmoid ? launch(moe_route_bwd_kernel<__nv_bfloat16, L, V, true>) : launch(moe_route_bwd_kernel<__nv_bfloat16, L, V, false>);
    else sigmoid ? launch(moe_route_bwd_kernel<float, L, V, true>) : launch(moe_route_bwd_kernel<float, L, V, false>);
    return cudaGetLastError() == cudaSuccess ? 0 : 4;
  });
}
