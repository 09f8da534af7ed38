// 16-bit operand times the values of an MXFP4 matrix, sm_100a: the gradient of a 4-bit product with respect to its activations.
//
//   C[g][M, K] = A[g][M, N] * values(B[g][N, K])      A bf16, B codes and scales with blocks along K, sums in fp32, C bf16 or fp32
//
// B is the weight as the forward product has it, so its values are written nowhere: a stage's codes (64 rows x 128 bytes) are turned into bf16 in shared
// memory, in the layout of an MN-major operand, and go from there to tcgen05.mma.  Against turning B into a bf16 matrix first that saves writing and reading
// it at 2 bytes a value (64 experts of 1408 x 2048: 740 MB), which is more than everything else of such a gradient over few rows.
//
// B takes the 128 rows of the MMA (twice: a tile has 256 columns of C), A's rows its N, up to 256 and a multiple of 16: an MMA's time is what it reads from
// shared memory, so that 160 rows cost 160 and not 256.  The two accumulators take all of TMEM where there are more than 128 rows, so that what is turned
// is used by as many rows as there may be; with fewer the next tile has accumulators of its own.
//
// Turning a stage takes eight warps some 900 cycles, most of them the arithmetic of the codes, and the MMAs 640 (160 rows); so two sets of eight warps take the
// stages in turn.  A set turns its first stage of the next tile before it reads out the last one, for the MMAs to go on as soon as they may.
// Measured: 64 experts of 1408 x 2048, 16 rows 54 us, 160 rows 70 (0.85 PFLOP/s; one set for all stages: 88), 1280 rows 424 (1.11).  Of a tile's 28000 cycles at
// 160 rows 14000 are MMAs, 6000 their wait for the accumulators to be stored - all SMs store at once, at 3.6 TB/s - and the rest what it takes to fill
// the rings again.  Values transposed on the way, for an operand that is K-major, take more instructions and are no faster (73 us); all of a warp's
// columns in registers before the first store would free the accumulators, but spill.
//   warp 0: TMA of A | warp 1: TMEM owner, MMAs | warp 2: TMA of codes and scales | warps 3..18: codes to values, and the tile's epilogue
#include <algorithm>

#include "mx4.cuh"

namespace apb {

constexpr int MV_SETS = 2, MV_SET_WARPS = 8, MV_WARPS = MV_SETS * MV_SET_WARPS, MV_FIRST_WARP = 3, MV_THREADS = 32 * (MV_FIRST_WARP + MV_WARPS);
constexpr int MV_BN = 64, MV_COLS = 256;  // rows of B in a stage, and columns of the tile
constexpr int MV_CODES = MV_BN * MX_ROW_BYTES, MV_SLOT = MV_BN * MV_COLS * 2;  // bytes of a stage: of codes, of values
// Rings of codes with their scales, of values, and of A in what is left, in stages of as many rows as the tile has.
constexpr int MV_C_RING = 4, MV_V_RING = 3, MV_A_MAX = 6;
static_assert(MV_C_RING % MV_SETS == 0, "a set meets every use of its slots of the codes");
constexpr int MV_A_BYTES = 227 * 1024 - 1024 - 256 - MV_C_RING * (MV_CODES + MX_SC_BYTES) - MV_V_RING * MV_SLOT;
constexpr int MV_SMEM = 227 * 1024;
static_assert(MV_A_BYTES >= 2 * 256 * MV_BN * 2, "two stages of A of a full tile");

struct MxValuesParams {
  GemmParams p;  // M, N = columns of C, ldc, out_fp32, status
  int tiles, m_tiles, stages;  // stages: of 64 along the contraction
  int rows, a_ring;            // rows of a tile, a multiple of 16; stages of A
};

// Codes at the bottoms of a word's halves, ``AT`` bits up, to a pair of bf16: sign, and e e m as the lowest bits of the exponent and the highest of the
// mantissa, which is the code's value * 2^-126 (0.5 as a denormal).  One multiplication moves both (the copies do not overlap), the rest is masked out.
template <int AT>
__device__ __forceinline__ uint32_t mx_two_bf16(uint32_t w) {
  return ((w & (0x000F000Fu << AT)) * (0x1040u >> AT)) & 0x81C081C0u;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__global__ void __launch_bounds__(MV_THREADS, 1)
gemm_mx4_values_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSB,
                       MxValuesParams q) {
  const GemmParams& p = q.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sB = smem;                           // [ring] codes: 64 rows of 128 bytes
  uint8_t* sSc = sB + MV_C_RING * MV_CODES;     // [ring of the codes] scales of 128 rows
  uint8_t* sV = sSc + MV_C_RING * MX_SC_BYTES;  // [ring] values: four chunks of 64 columns, 64 rows of 128 bytes each
  uint8_t* sA = sV + MV_V_RING * MV_SLOT;       // [ring] a tile's rows of 128 bytes
  uint64_t* bars = reinterpret_cast<uint64_t*>(sA + MV_A_BYTES);
  uint64_t *a_full = bars, *a_empty = a_full + MV_A_MAX, *c_full = a_empty + MV_A_MAX, *c_empty = c_full + MV_C_RING, *turned = c_empty + MV_C_RING,
           *used = turned + MV_V_RING, *acc_full = used + MV_V_RING, *acc_free = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  constexpr int CHUNK_BYTES = MV_BN * 128;
  static_assert((2 * (MV_A_MAX + MV_C_RING + MV_V_RING) + 4) * 8 + 8 <= 256, "barrier block");
  static_assert(MV_C_RING * MX_SC_BYTES % 1024 == 0, "alignment of swizzled slots");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MV_A_MAX; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], 1);
    }
    for (int s = 0; s < MV_C_RING; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], MV_SET_WARPS);
    }
    for (int s = 0; s < MV_V_RING; ++s) {
      mbar_init(&turned[s], MV_SET_WARPS);
      mbar_init(&used[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_free[b], MV_WARPS);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_previous();

  auto fail = [&](uint32_t code) {
    atomicCAS(p.status, 0u, code);
    *abort_flag = 1;
  };
  // tile -> group, rows, columns; the row tiles of a column tile come one after the other: its codes are in L2 then
  auto place = [&](int t, int& grp, int& m0, int& col) {
    grp = p.div_tiles.div(t);
    const int r = t - grp * (int)p.div_tiles.d, tn = p.div_group.div(r);
    m0 = (r - tn * q.m_tiles) * q.rows;
    col = tn * MV_COLS;
  };
  const int a_bytes = q.rows * MV_BN * 2;
  const int bufs = q.rows <= 128 ? 2 : 1;  // accumulators of two tiles, 128 columns apart, or of one
  if (warp == 0) {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x) {
        int grp, m0, col;
        place(t, grp, m0, col);
        for (int k = 0; k < q.stages; ++k) {
          if (!mbar_wait(&a_empty[slot], phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_EMPTY);
            break;
          }
          mbar_expect_tx(&a_full[slot], a_bytes);
          tma_load_3d(sA + slot * a_bytes, &tmA, &a_full[slot], k * MV_BN, m0, grp);
          if (++slot == q.a_ring) slot = 0, phase ^= 1;
        }
      }
      let_next_in();
    }
  } else if (warp == 2) {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x) {
        int grp, m0, col;
        place(t, grp, m0, col);
        for (int k = 0; k < q.stages; ++k) {
          if (!mbar_wait(&c_empty[slot], phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_EMPTY);
            break;
          }
          mbar_expect_tx(&c_full[slot], MV_CODES + MX_SC_BYTES);
          tma_load_3d(sB + slot * MV_CODES, &tmB, &c_full[slot], col / 2, k * MV_BN, grp);
          tma_load_3d(sSc + slot * MX_SC_BYTES, &tmSB, &c_full[slot], col / MX_BK * (MX_SC_BYTES / 4), k * MV_BN / 128, grp);
          if (++slot == MV_C_RING) slot = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t a_desc = make_smem_desc(smem_u32(sA), 16, 1024), v_desc = make_smem_desc(smem_u32(sV), CHUNK_BYTES, 1024);
      int a_slot = 0, v_slot = 0;
      uint32_t a_phase = 0, v_phase = 0, seq = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x, ++seq) {
        int grp, m0, col;
        place(t, grp, m0, col);
        const uint32_t idesc = make_idesc_bf16(128, (min(p.M - m0, q.rows) + 15) / 16 * 16, 1, 0);
        const uint32_t buf = bufs == 2 ? seq & 1u : 0u, turn = bufs == 2 ? seq >> 1 : seq, d_tmem = tmem + 128 * buf;
        if (turn > 0 && !mbar_wait(&acc_free[buf], (turn - 1) & 1, abort_flag)) {
          fail(ST_TIMEOUT_TMEM_EMPTY);
          break;
        }
        tc_fence_after();
        for (int k = 0; k < q.stages; ++k) {
          if (!mbar_wait(&a_full[a_slot], a_phase, abort_flag) || !mbar_wait(&turned[v_slot], v_phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_FULL);
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < MV_BN / UMMA_K; ++kk) {
            const uint64_t ad = a_desc + desc_offset(a_slot * a_bytes + kk * UMMA_K * 2), vd = v_desc + desc_offset(v_slot * MV_SLOT + kk * UMMA_K * 128);
            const uint32_t more = k > 0 || kk > 0 ? 1u : 0u;
            umma_f16(d_tmem, vd, ad, idesc, more);
            umma_f16(d_tmem + 256, vd + desc_offset(MV_SLOT / 2), ad, idesc, more);
          }
          umma_commit(&a_empty[a_slot]);
          umma_commit(&used[v_slot]);
          if (++a_slot == q.a_ring) a_slot = 0, a_phase ^= 1;
          if (++v_slot == MV_V_RING) v_slot = 0, v_phase ^= 1;
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
    }
  } else {
    const int w = warp - MV_FIRST_WARP, set = w / MV_SET_WARPS, quarter = warp & 3, half = w / 4 % 2;
    // A warp turns eight rows of a stage, a lane two blocks of 32 columns of one: eight lanes on eight rows, so that neither the swizzled codes nor the
    // values meet in a bank.  Of eight columns, which are a word of codes, column j comes into the low half of word j or the high half of word j - 4: the
    // tensor cores do not care, and the epilogue has every lane's column.
    const int row = w % MV_SET_WARPS * 8 + (lane & 7), block = lane >> 3, swizzle = lane & 7;
    const uint32_t from = row * 128 + ((block ^ swizzle) << 4), from2 = row * 128 + (((block + 4) ^ swizzle) << 4);  // bytes of a stage's codes
    const uint32_t to = (block >> 1) * CHUNK_BYTES + row * 128, unit = ((block & 1) * 4) ^ swizzle;                   // and of its values
    auto turn_stage = [&](const uint8_t* codes, const uint8_t* sc, uint8_t* values) {
      const uint4 c[2] = {*reinterpret_cast<const uint4*>(codes + from), *reinterpret_cast<const uint4*>(codes + from2)};
      const uint32_t e[2] = {sc[0], sc[MX_SCALE_TILE]};
      // 2^-126 goes with the scale, in one multiplication, where the product is a bf16: scales up to 2, which is every weight below 16
      const bool plain = __all_sync(0xffffffffu, max(e[0], e[1]) <= 128u);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t x[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
        const uint32_t scale = (plain ? (e[i] + 126u) << 7 : e[i] == 255u ? 0x7FC0u : e[i] == 0u ? 0x0040u : e[i] << 7) * 0x10001u;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t y = x[u] >> 8;
          uint32_t r[4] = {mx_two_bf16<0>(x[u]), mx_two_bf16<4>(x[u]), mx_two_bf16<0>(y), mx_two_bf16<4>(y)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!plain) r[j] = mul_bf16x2(r[j], 0x7E807E80u);  // 2^126
            r[j] = mul_bf16x2(r[j], scale);
          }
          *reinterpret_cast<uint4*>(values + to + i * 2 * CHUNK_BYTES + ((unit ^ u) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
        }
      }
    };
    // Accumulators to C.  A warp has 32 columns of C in its TMEM lanes, half of a set's warps in the one accumulator and half in the other; A's rows are
    // TMEM columns, 32 at a time, which the sets take in turn.  A store of a warp is 64 or 128 bytes of a row.
    auto epilogue = [&](int t, uint32_t seq) {
      const uint32_t buf = bufs == 2 ? seq & 1u : 0u, turn = bufs == 2 ? seq >> 1 : seq;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], turn & 1u, abort_flag))) {
        fail(ST_TIMEOUT_TMEM_FULL);
        return false;
      }
      tc_fence_after();
      int grp, m0, col;
      place(t, grp, m0, col);
      const int rows = min(p.M - m0, q.rows), esz = p.out_fp32 ? 4 : 2;
      const int column = col + 128 * half + 32 * quarter + (lane & ~7) + (lane >> 1 & 3) + (lane & 1) * 4;
      const bool in = column < p.N;
      const long long step = p.ldc * esz;
      uint8_t* C = reinterpret_cast<uint8_t*>(p.C) + (((long long)grp * p.M + m0) * p.ldc + column) * esz;
#pragma unroll 1
      for (int m = 32 * set; m < rows; m += 32 * MV_SETS) {
        uint32_t r[32];
        tmem_ld_32x32(tmem + (uint32_t(quarter * 32) << 16) + 128 * buf + 256 * half + m, r);
        tmem_ld_wait_for(r);
        uint8_t* dst = C + m * step;
#pragma unroll
        for (int i = 0; i < 32; ++i, dst += step) {
          if (!in || m + i >= rows) continue;
          if (p.out_fp32) *reinterpret_cast<uint32_t*>(dst) = r[i];
          else *reinterpret_cast<__nv_bfloat16*>(dst) = __float2bfloat16(__uint_as_float(r[i]));
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_free[buf]);
      return true;
    };
    int c_slot = 0, v_slot = 0, last = -1;  // last: a tile that is still to be read out, ``seq`` - 1 of this CTA
    uint32_t c_phase = 0, v_phase = 1, it = 0, seq = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x, ++seq) {
      int grp, m0, col;
      place(t, grp, m0, col);
      for (int k = 0; k < q.stages && ok; ++k, ++it) {
        if ((int)(it % MV_SETS) == set) {
          ok = __all_sync(0xffffffffu, mbar_wait(&c_full[c_slot], c_phase, abort_flag) && mbar_wait(&used[v_slot], v_phase, abort_flag));
          if (!ok) {
            fail(ST_TIMEOUT_FULL);
            break;
          }
          turn_stage(sB + c_slot * MV_CODES, sSc + c_slot * MX_SC_BYTES + mx_scale_at((k * MV_BN + row) & 127, block), sV + v_slot * MV_SLOT);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&turned[v_slot]);
            mbar_arrive(&c_empty[c_slot]);
          }
          if (last >= 0) {
            ok = epilogue(last, seq - 1);
            last = -1;
          }
        }
        if (++c_slot == MV_C_RING) c_slot = 0, c_phase ^= 1;
        if (++v_slot == MV_V_RING) v_slot = 0, v_phase ^= 1;
      }
      if (ok && last >= 0) ok = epilogue(last, seq - 1);  // (a tile of one stage, which was the other set's)
      last = t;
    }
    if (ok && last >= 0) epilogue(last, seq - 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace apb

using namespace apb;

extern "C" int apb_gemm_get_reserved_sms();

// Whether this kernel is the better choice against the values as a matrix of their own and the 16-bit product: with few rows, where the matrix is most of
// what is moved, and tiles for every SM.  us, this / that: 64 experts of 1408 x 2048, 16 rows 54 / 146, 160 rows 70 / 165, 1280 rows 424 / 385; 16 of 2048 x
// 2048, 512 rows 71 / 85; one of 4096 x 4096, 128 rows (16 tiles) 45 / 20, 2048 rows (128 tiles) 54 / 54, of 4096 x 14336, 1024 rows 103 / 104, of 14336 x
// 4096, 16 rows (16 tiles) 117 / 49.  Its CTAs take an SM's registers, so that it is not taken where room for communication kernels is asked for.
extern "C" int apb_gemm_mx4_values_takes(long long G, long long M, long long K, int num_sms) {
  return !apb_gemm_makes_room() && M <= 512 && G * ((M + 255) / 256) * ((K + MV_COLS - 1) / MV_COLS) >= num_sms;
}

// A [G, M, N] bf16 (N % 8 == 0), B codes [G, N, kp / 2] and SB, C [G, M, K]; all dense, 16-byte bases.
// Returns 0, or an argument / driver / launch error (nothing launched; 3: not this kernel's form).
extern "C" int apb_gemm_mx4_values(const void* A, const void* B, const void* SB, void* C, long long G, long long M, long long N, long long K, int out_fp32,
                                   uint32_t* status, int num_sms, cudaStream_t stream) {
  const long long kp = (K + 31) / 32 * 32;
  if (G < 0 || M < 0 || N < 0 || K < 0 || M >= 1ll << 30 || N >= 1ll << 30 || K >= 1ll << 30 || N % 8) return 3;
  if (G == 0 || M == 0 || K == 0) return 0;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(SB) | reinterpret_cast<uintptr_t>(C)) & 15) return 3;
  if (N == 0) return zero_result(C, G * M, K, K, out_fp32, stream);
  MxValuesParams q{};
  GemmParams& p = q.p;
  p.M = (int)M;
  p.N = (int)K;
  p.C = C;
  p.ldc = K;
  p.out_fp32 = out_fp32;
  p.status = status;
  q.m_tiles = (int)((M + 255) / 256);
  q.rows = (int)(((M + q.m_tiles - 1) / q.m_tiles + 15) / 16 * 16);
  q.a_ring = std::min(MV_A_MAX, MV_A_BYTES / (q.rows * MV_BN * 2));
  q.stages = (int)((N + MV_BN - 1) / MV_BN);
  const long long n_tiles = (K + MV_COLS - 1) / MV_COLS, tiles = G * q.m_tiles * n_tiles;
  if (tiles >= 1ll << 30) return 3;
  q.tiles = (int)tiles;
  p.div_tiles = FastDiv((uint32_t)(q.m_tiles * n_tiles));
  p.div_group = FastDiv((uint32_t)q.m_tiles);
  CUtensorMap tmA, tmB, tmSB;
  int e = make_map_3d(&tmA, A, (uint64_t)N, (uint64_t)M, (uint64_t)G, (uint64_t)N, (uint32_t)q.rows);
  if (!e) e = mx_map(&tmB, B, kp / 2, N, G, MX_ROW_BYTES, MV_BN, false);
  if (!e) e = mx_map(&tmSB, SB, (uint64_t)((kp + 127) / 128) * (MX_SCALE_TILE / 4), (N + 127) / 128, G, MX_SC_BYTES / 4, 1, true);
  if (e) return e;
  const int usable = std::max(1, num_sms - apb_gemm_get_reserved_sms());
  cudaFuncSetAttribute(gemm_mx4_values_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MV_SMEM);
  launch_after(gemm_mx4_values_kernel, (unsigned)std::min(q.tiles, usable), MV_THREADS, MV_SMEM, stream, tmA, tmB, tmSB, q);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
