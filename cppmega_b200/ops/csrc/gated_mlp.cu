// Gated feed-forward block on CTA pairs: y = (act(x Wg^T) * (x Wu^T)) W2^T with w1 = [Wg; Wu].
//   gated_kernel, forward   one product with both projections: a tile of 256 tokens holds the same columns of gate and up side by side
//                           in TMEM, the epilogue forms h = act(g) u from the fp32 accumulators and stores h and, for training, g and u.
//   gated_kernel, backward  dh = dy W2 stays in TMEM; the epilogue reads g and u and stores dg = dh u act'(g), du = dh act(g).
// The other products (h W2^T, [dg du] w1, [dg du]^T x, dy^T h) are dense ones, with the last wave shared (gemm_split.cu).  Against linear,
// activation, linear this saves writing and reading dh, reading [g u] in the forward, and two launches.  Bound by the tensor cores:
// 4096 x 3584 x 18944 forward 714 us at 95 % of the tensor pipe, backward 396 us at 91 % (at the clocks of a loop).
//
// Both kernels are the 256 x 256 x 64 tcgen05.mma.cta_group::2 pipeline of gemm_pair.cu (6 or 5 stages of 32 KB, two accumulators in TMEM,
// every wait bounded, no multicast).  The first CTA of a pair loads the gate rows of w1 and the second the up rows, so that the tile is
// one ordinary 256-column product.  The epilogue has eight warps, two to a TMEM quadrant: its exponentials, and in the backward its
// loads of g and u, have to fit under the main loop of the next tile.
//
// Few tokens (serving): both products read their weights once through few_rows.cu; the sums of the first one's partial tiles, the
// activation and the product are one small kernel, the sums of the second another.
#include <cuda_fp16.h>

#include "few_rows.cuh"
#include "fp32_pair.cuh"
#include "gemm_split.cuh"
#include "pair_issue.cuh"

namespace cm {
namespace mlp {

using namespace pair2;

constexpr int BM = 128;                 // rows of one CTA; a tile has 2 * BM
constexpr int BK = 64;
constexpr int UMMA_K = 16;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int A_BYTES = BM * BK * 2;
constexpr int STAGE_BYTES = 2 * A_BYTES;
constexpr int STORE_BYTES = 32 * 64;    // one warp's 32 rows x 32 columns of 16-bit values
constexpr int STORE_BUFS = 2;
// Shared memory: operand stages, store staging, and with INBOX one chunk of g and u per epilogue warp on its way in.
template <bool INBOX>
struct Smem {
  static constexpr int STAGES = INBOX ? 5 : 6;
  static constexpr int FETCH_BYTES = INBOX ? 2 * STORE_BYTES : 0;
  static constexpr int STORE_OFF = STAGES * STAGE_BYTES;
  static constexpr int FETCH_OFF = STORE_OFF + EPI_WARPS * STORE_BUFS * STORE_BYTES;
  static constexpr int BAR_OFF = FETCH_OFF + EPI_WARPS * FETCH_BYTES;
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;
};
static_assert(Smem<true>::TOTAL <= 227 * 1024 && Smem<false>::TOTAL <= 227 * 1024, "shared memory of a block");

enum Act : int { SILU = 0, GELU_TANH = 1, RELU = 2 };

// g and u are kept for the backward as 16-bit floats of 11 bits under one power of two per row and 32 columns: as bf16 they would bring a
// third rounding of 2^-9 into dx and dw1, next to those of the products' operands and of the results (3.0e-3 against 2.4e-3 of the
// gradients' norm).  The largest value of a group lies in [2^14, 2^15); what is 2^29 times smaller loses bits, and nothing overflows.  Of a
// gate that is closed, far out on its negative side, the size has no part in any gradient: it counts as closed_at, beyond which act and its
// slope are zero in fp32, so that it does not take its neighbours' bits, and is kept as the lowest fp16 number where it has no room.
//   kept = [M][2F] fp16 (g, then u), then [2][groups][M] bytes: the exponent field of the power that the values were multiplied with
struct Kept {
  __half* v;
  uint8_t* power;
  long long plane;        // bytes between the powers of g and of u
  __host__ __device__ static long long groups(int F) { return (F + 31) / 32; }
  __host__ __device__ static long long bytes(long long M, int F) { return 4 * M * F + 2 * groups(F) * M; }
  __host__ static Kept at(void* p, long long M, int F) {
    return Kept{static_cast<__half*>(p), static_cast<uint8_t*>(p) + 4 * M * F, groups(F) * M};
  }
};
// exponent field of the power for a group whose largest magnitude is m; 253 at most, so that its inverse is a normal number
__device__ __forceinline__ uint32_t power_for(float m) { return min(268u - (__float_as_uint(m) >> 23), 253u); }
__device__ __forceinline__ float power_of(uint32_t field) { return __uint_as_float(field << 23); }
__device__ __forceinline__ float inverse_power(uint32_t field) { return __uint_as_float((254u - field) << 23); }

struct Args {
  int M, F, K;            // tokens, ffn columns, reduction (hidden)
  int bn;                 // accumulator columns of a tile: 256 or 128
  Kept kept;              // v null: not kept
  int* err;
};

// act(g), and its slope, for two values at a time: the epilogues have two warps a scheduler, and their instructions are what a tile with a
// short main loop waits for.  The logistic function's approximations err by a few 2^-24, which vanishes in the bf16 results.
constexpr float GELU_C = 0.7978845608028654f, GELU_K = 0.044715f;      // sqrt(2 / pi); (1 + tanh t) / 2 = sigmoid(2 t)
__device__ __forceinline__ Pair relu_of(Pair g) {
  const float2 f = pr_get(g);
  return pr(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);             // NaN stays
}
template <int ACT>
__device__ __forceinline__ Pair act_of(Pair g) {
  if constexpr (ACT == RELU) return relu_of(g);
  if constexpr (ACT == SILU) return g * sigmoid_of(g);
  return g * sigmoid_of(g * pr_fma(g * g, pr(2.f * GELU_C * GELU_K), pr(2.f * GELU_C)));
}
template <int ACT>
__device__ __forceinline__ float act_of(float g) {
  return pr_get(act_of<ACT>(pr(g))).x;
}
template <int ACT>
__device__ __forceinline__ void act_slope(Pair g, Pair& a, Pair& slope) {
  if constexpr (ACT == RELU) {
    const float2 f = pr_get(g);
    a = relu_of(g);
    slope = pr(f.x > 0.f ? 1.f : 0.f, f.y > 0.f ? 1.f : 0.f);
  } else if constexpr (ACT == SILU) {
    const Pair q = sigmoid_of(g);
    a = g * q;
    slope = pr_fma(a, pr_fma(pr(-1.f), q, pr(1.f)), q);                // q + g q (1 - q)
  } else {
    const Pair q = sigmoid_of(g * pr_fma(g * g, pr(2.f * GELU_C * GELU_K), pr(2.f * GELU_C)));
    a = g * q;
    const float2 f = pr_get(g);                                        // far out q or 1 - q is 0, and the factor must not be infinite
    const Pair b = pr(fminf(fmaxf(f.x, -1e6f), 1e6f), fminf(fmaxf(f.y, -1e6f), 1e6f));
    const Pair inner = b * pr_fma(b * b, pr(6.f * GELU_C * GELU_K), pr(2.f * GELU_C));
    slope = pr_fma(q * pr_fma(pr(-1.f), q, pr(1.f)), inner, q);        // q + q (1 - q) b 2 c (1 + 3 k b^2)
  }
}

// What a gate counts for in its group's power of two.
template <int ACT>
__device__ __forceinline__ float gate_size(float g) {
  constexpr float closed_at = ACT == RELU ? 0.f : -128.f;
  return fabsf(fmaxf(g, closed_at));
}
__device__ __forceinline__ uint32_t saturated_half2(float lo, float hi) {
  uint32_t p;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
  return p;
}

// values 2 j and 2 j + 1 of an accumulator's row; two values as bf16
__device__ __forceinline__ Pair two(const uint32_t (&v)[32], int j) { return pr(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])); }
__device__ __forceinline__ uint32_t bf16_of(Pair p) {
  const float2 f = pr_get(p);
  return pack_bf16(f.x, f.y);
}

// A warp's 32 rows x 32 columns on their way out: a ring of staging buffers (64-byte swizzle), each left by one bulk tensor store.
struct Outbox {
  uint8_t* base;
  int lane;
  uint32_t at = 0;
  __device__ __forceinline__ void put(const CUtensorMap* map, const uint32_t (&v)[16], int col, int row) {
    uint8_t* buf = base + at * STORE_BYTES;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(STORE_BUFS - 1) : "memory");   // this buffer has been read
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      bulk_store_2d(map, buf, col, row);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    at = at + 1 == STORE_BUFS ? 0 : at + 1;
  }
};

// BACK = false: A = x, B = w1 (rows of g and u), outputs h (tmO0), g (tmO1), u (tmO2).
// BACK = true:  A = dy, B = w2 (reduction rows), outputs dg (tmO1), du (tmO2).
template <bool BACK, int ACT, bool INBOX>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gated_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmO0,
             const __grid_constant__ CUtensorMap tmO1, const __grid_constant__ CUtensorMap tmO2, const Args args) {
  using S = Smem<INBOX>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  // the dynamic segment starts at the same offset in both CTAs, so the aligned offsets agree as the descriptors need
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int half = args.bn >> 1;
  const int cols = BACK ? args.bn : half;                       // ffn columns of a tile
  const int tiles_n = (args.F + cols - 1) / cols, tiles_m = (args.M + 2 * BM - 1) / (2 * BM), total = tiles_m * tiles_n;
  const int nkb = (args.K + BK - 1) / BK;
  const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;
  // bands of 8 row tiles, as in gemm_pair.cu: the tiles in flight share their operands in L2
  auto place = [&](int tile, int& m0, int& n0) {
    const int band_tiles = 8 * tiles_n, b = tile / band_tiles, in = tile - b * band_tiles, rows = min(8, tiles_m - b * 8);
    m0 = (b * 8 + in % rows) * 2 * BM;
    n0 = (in / rows) * cols;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], 2 * EPI_WARPS);
    }
    *abort_flag = (args.err && *reinterpret_cast<volatile int*>(args.err) != 0) ? 1 : 0;   // an earlier kernel gave up: drain
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------ TMA producer (both CTAs) ------------------------------
    if (elect_one()) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      const uint32_t pair_bytes = 2 * (A_BYTES + half * 128);
      uint32_t stage = 0, phase = 0, used = 0;
      bool ok = *abort_flag == 0;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        int m0, n0;
        place(tile, m0, n0);
        const int ma = m0 + rank * BM, nb = BACK ? n0 + rank * half : n0 + rank * args.F;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, args.err, ERR_WAIT_EMPTY);
          if (!ok) break;
          uint8_t* sa = smem + stage * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          if (rank == 0) mbar_expect_tx(&full_bar[stage], pair_bytes);
          const uint32_t bar = map_to_rank(smem_u32(&full_bar[stage]), 0);
          const int k0 = kb * BK;
          load_2d(sa, &tmA, bar, k0, ma);                                                // box [128 rows, 64 k]
          if (!BACK) {
            load_2d(sb, &tmB, bar, k0, nb);                                              // box [half rows, 64 k]
          } else {
            for (int c = 0; c < half / 64; ++c) load_2d(sb + c * (BK * 128), &tmB, bar, nb + c * 64, k0);   // boxes [64 k, 64 n]
          }
          if (used < STAGES) ++used;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // the last releases of this CTA's stages come from the partner: see them arrive before the barriers go away
      for (uint32_t i = 0; i < used && ok; ++i) {
        const uint32_t s = (stage + STAGES - 1 - i) % STAGES;
        const uint32_t ph = (stage >= i + 1) ? phase : phase ^ 1;
        ok = mbar_wait(&empty_bar[s], ph, abort_flag, args.err, ERR_WAIT_EMPTY);
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (first CTA) ------------------------------
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = umma_idesc_bf16(2 * BM, args.bn, false, BACK);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = *abort_flag == 0;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        ok = mbar_wait(&tmem_empty[acc], acc_phase ^ 1, abort_flag, args.err, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, abort_flag, args.err, ERR_WAIT_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
          const uint32_t sb = sa + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t ad = umma_desc_sw128(sa + k * (UMMA_K * 2), 16, 1024);
            const uint64_t bd = BACK ? umma_desc_sw128(sb + k * (UMMA_K * 128), BK * 128, 1024) : umma_desc_sw128(sb + k * (UMMA_K * 2), 16, 1024);
            mma_2cta(d_tmem, ad, bd, idesc, (kb | k) != 0);
          }
          commit_pair(&empty_bar[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        commit_pair(&tmem_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    // ------------------------------ epilogue (both CTAs) ------------------------------
    const int q = warp & 3;                                     // TMEM lane quadrant this warp may read
    const int part = (warp - 2) >> 2;                           // which half of the tile's columns
    Outbox out{smem + S::STORE_OFF + (warp - 2) * STORE_BUFS * STORE_BYTES, lane};
    const int c_begin = part * (cols >> 1), c_end = c_begin + (cols >> 1);
    // Backward: g and u of the chunks (32 rows x 32 columns) of this warp's tiles are requested in the order in which they are needed and
    // one ahead, over the ends of tiles too: a row to a lane into registers, or with INBOX a row to four lanes into shared memory (64-byte
    // swizzle, as in the Outbox), where an instruction touches 8 lines instead of 32.  Past the last row or column come zeros.
    uint8_t* inbox = smem + S::FETCH_OFF + (warp - 2) * S::FETCH_BYTES;
    int ahead_tile = first_tile, ahead_c = c_begin;
    uint32_t powers = 0;                                        // of the chunk on its way: g's, u's << 8
    uint4 gv[4], uv[4];                                         // the chunk on its way, without INBOX
    auto fetch = [&]() {
      if (ahead_tile < total) {
        int m0, n0;
        place(ahead_tile, m0, n0);
        const int base = m0 + rank * BM + q * 32, col = n0 + ahead_c;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int r = INBOX ? v * 8 + (lane >> 2) : lane, piece = INBOX ? lane & 3 : v;
          const bool on = base + r < args.M && col + 8 * piece < args.F;
          const __half* p = on ? args.kept.v + (long long)(base + r) * 2 * args.F + col + 8 * piece : args.kept.v;
          if constexpr (INBOX) {
            const uint32_t dst = smem_u32(inbox + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(on ? 16 : 0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + STORE_BYTES), "l"(on ? p + args.F : p), "r"(on ? 16 : 0)
                         : "memory");
          } else {
            gv[v] = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            uv[v] = on ? *reinterpret_cast<const uint4*>(p + args.F) : make_uint4(0, 0, 0, 0);
          }
        }
        powers = 127u | 127u << 8;
        if (base + lane < args.M && col < args.F) {
          const uint8_t* e = args.kept.power + (long long)(col >> 5) * args.M + base + lane;
          powers = uint32_t(e[0]) | uint32_t(e[args.kept.plane]) << 8;
        }
        ahead_c += 32;
        if (ahead_c == c_end) { ahead_c = c_begin; ahead_tile += tile_step; }
      }
      if constexpr (INBOX) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t acc = 0, acc_phase = 0;
    bool ok = *abort_flag == 0;
    if constexpr (BACK) fetch();
    for (int tile = first_tile; tile < total && ok; tile += tile_step) {
      int m0, n0;
      place(tile, m0, n0);
      const int row0 = m0 + rank * BM + q * 32, row = row0 + lane;
      ok = __all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, abort_flag, args.err, ERR_WAIT_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_base = tmem_base + acc * 256 + (uint32_t(q * 32) << 16);
      if constexpr (!BACK) {
        if (row0 < args.M) {
          for (int c = c_begin; c < c_end && n0 + c < args.F; c += 32) {
            uint32_t g[32], u[32];
            tmem_ld_32x32(t_base + c, g);
            tmem_ld_32x32(t_base + half + c, u);
            tmem_ld_wait();
            uint32_t o[16];
            if (args.kept.v) {
              auto keep = [&](const uint32_t (&v)[32], auto size, const CUtensorMap* map, uint8_t* power) {
                float m = 0.f;
                if (n0 + c + 32 <= args.F) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) m = fmaxf(m, size(__uint_as_float(v[j])));
                } else {                                        // the gate's columns past the last are up's first rows: not of this group
#pragma unroll
                  for (int j = 0; j < 32; ++j)
                    if (n0 + c + j < args.F) m = fmaxf(m, size(__uint_as_float(v[j])));
                }
                const uint32_t field = power_for(m);
                const float k = power_of(field);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  const float2 f = pr_get(two(v, j) * pr(k));
                  o[j] = saturated_half2(f.x, f.y);
                }
                out.put(map, o, n0 + c, row0);
                if (row < args.M) power[(long long)((n0 + c) >> 5) * args.M + row] = uint8_t(field);
              };
              keep(g, gate_size<ACT>, &tmO1, args.kept.power);
              keep(u, [](float v) { return fabsf(v); }, &tmO2, args.kept.power + args.kept.plane);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = bf16_of(act_of<ACT>(two(g, j)) * two(u, j));
            out.put(&tmO0, o, n0 + c, row0);
          }
        }
      } else {
#pragma unroll 1
        for (int c = c_begin; c < c_end; c += 32) {
          const bool any = row0 < args.M && n0 + c < args.F;     // the same in all lanes
          uint32_t d[32];
          if (any) tmem_ld_32x32(t_base + c, d);
          if constexpr (INBOX) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
          }
          uint4 gc[4], uc[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int at = lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4);
            gc[v] = INBOX ? *reinterpret_cast<const uint4*>(inbox + at) : gv[v];
            uc[v] = INBOX ? *reinterpret_cast<const uint4*>(inbox + STORE_BYTES + at) : uv[v];
          }
          const float gi = inverse_power(powers & 255u), ui = inverse_power(powers >> 8);
          if constexpr (INBOX) __syncwarp();                     // read by every lane: the next chunk may come
          fetch();
          if (!any) continue;
          tmem_ld_wait();
          uint32_t og[16], ou[16];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const __half2* gb = reinterpret_cast<const __half2*>(&gc[v]);
            const __half2* ub = reinterpret_cast<const __half2*>(&uc[v]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 g = __half22float2(gb[j]), u = __half22float2(ub[j]);
              Pair a, slope;
              act_slope<ACT>(pr(g.x, g.y) * pr(gi), a, slope);
              const Pair dh = two(d, 4 * v + j);
              og[4 * v + j] = bf16_of(dh * (pr(u.x, u.y) * pr(ui)) * slope);
              ou[4 * v + j] = bf16_of(dh * a);
            }
          }
          out.put(&tmO1, og, n0 + c, row0);
          out.put(&tmO2, ou, n0 + c, row0);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&tmem_empty[acc]), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if constexpr (INBOX) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // ------------------------------ teardown ------------------------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // let TMA copies and MMAs still in flight land before the pair's shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
    __syncthreads();
  }
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// A [rows, cols] result with row pitch ld as the target of bulk stores: boxes of 32 rows x 32 columns.
static int make_out_map(CUtensorMap* out, void* base, long long rows, long long cols, long long ld) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return -1;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {32, 32}, one[2] = {1, 1};
  CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

template <bool BACK, int ACT, bool INBOX>
static int launch(const CUtensorMap* maps, const Args& args, cudaStream_t stream) {
  auto kern = gated_kernel<BACK, ACT, INBOX>;
  static PerDevice configured;
  if (configured.first()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<INBOX>::TOTAL) != cudaSuccess) return -2;
    configured.done();
  }
  const int cols = BACK ? args.bn : args.bn / 2;
  const long long tiles = (long long)((args.M + 2 * BM - 1) / (2 * BM)) * ((args.F + cols - 1) / cols);
  if (tiles > 0x7fffffff) return -10;
  const int pairs = sm_count() / 2;
  const int grid = 2 * int(tiles < pairs ? tiles : pairs);
  kern<<<grid, THREADS, Smem<INBOX>::TOTAL, stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], args);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// Up to this reduction the backward's epilogue is longer than a tile's main loop, and g and u come through shared memory; above it the main
// loop is, and the operand stage that this costs counts more.  Registers against shared memory, us: 4096 x 512 x 8192 97 / 79, 16384 x 1024 x
// 2048 101 / 85, 16384 x 1536 x 2048 109 / 93, 8192 x 2048 x 2048 70 / 64; 8192 x 3584 x 2048 96 / 97, 4096 x 4096 x 21504 501 / 509,
// 100 x 4096 x 4096 23.3 / 24.5.
constexpr int INBOX_K = 2560;
template <bool BACK, int ACT>
static int launch_in(const CUtensorMap* maps, const Args& args, cudaStream_t stream) {
  if constexpr (BACK) {
    if (args.K <= INBOX_K) return launch<true, ACT, true>(maps, args, stream);
  }
  return launch<BACK, ACT, false>(maps, args, stream);
}

template <bool BACK>
static int launch_act(int act, const CUtensorMap* maps, const Args& args, cudaStream_t stream) {
  switch (act) {
    case SILU: return launch_in<BACK, SILU>(maps, args, stream);
    case GELU_TANH: return launch_in<BACK, GELU_TANH>(maps, args, stream);
    case RELU: return launch_in<BACK, RELU>(maps, args, stream);
  }
  return -10;
}

// Accumulator columns of a tile: waves of pairs, weighted as in plan_dense (a 128-column tile takes 0.74 of a 256-column one's time).
static int plan_bn(int M, int F, bool back) {
  const long long pairs = sm_count() / 2, tm = (M + 2 * BM - 1) / (2 * BM);
  auto waves = [&](int bn) {
    const int cols = back ? bn : bn / 2;
    return (tm * ((F + cols - 1) / cols) + pairs - 1) / pairs;
  };
  return waves(128) * 17.8 < waves(256) * 24.2 ? 128 : 256;
}

// ------------------------------ few tokens ------------------------------
// A tile's sum over its partial tiles, for TOKS tokens of one weight row: their loads are in flight together, and the place of a partial
// tile is found once for all of them.  A long reduction over few tiles leaves dozens of partial tiles; blockDim.y threads then share them
// (first + y, first + y + blockDim.y, ...) and their sums are added in that order.
constexpr int TOKS = 8, MAX_SHARE = 8;
struct FewSums {
  float s[MAX_SHARE - 1][TOKS][few::TILE];
};
// The sums of NR weight rows at once, so that their loads are in flight together as well.
template <int NR>
__device__ __forceinline__ void few_sum(const float* __restrict__ part, const few::Cut& cut, const int (&row)[NR], int tok0, FewSums* share,
                                        float (&s)[NR][TOKS]) {
  const int n = cut.tokens - tok0;
  int tile[NR], c[NR], end[NR], left = 0;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    tile[r] = row[r] / few::TILE;
    c[r] = cut.first(tile[r]) + threadIdx.y;
    end[r] = cut.last(tile[r]);
    left = max(left, end[r] - c[r] + 1);
#pragma unroll
    for (int j = 0; j < TOKS; ++j) s[r][j] = 0.f;
  }
  for (; left > 0; left -= blockDim.y) {
    float v[NR][TOKS];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float* p = part + cut.at(c[r], tile[r]) + tok0 * few::TILE + row[r] % few::TILE;
      const bool on = c[r] <= end[r];
      if (n >= TOKS) {
#pragma unroll
        for (int j = 0; j < TOKS; ++j) v[r][j] = on ? p[j * few::TILE] : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < TOKS; ++j) v[r][j] = on && j < n ? p[j * few::TILE] : 0.f;
      }
      c[r] += blockDim.y;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int j = 0; j < TOKS; ++j) s[r][j] += v[r][j];
  }
  if (blockDim.y == 1) return;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (threadIdx.y > 0) {
#pragma unroll
      for (int j = 0; j < TOKS; ++j) share->s[threadIdx.y - 1][j][threadIdx.x] = s[r][j];
    }
    __syncthreads();
    if (threadIdx.y == 0) {
      for (int y = 1; y < blockDim.y; ++y)
#pragma unroll
        for (int j = 0; j < TOKS; ++j) s[r][j] += share->s[y - 1][j][threadIdx.x];
    }
    __syncthreads();
  }
}
// threads that share a tile's partial tiles
static int few_share(const few::Cut& c) {
  const int most = c.nkb / c.q + 2;
  return most <= 4 ? 1 : most <= 16 ? 4 : MAX_SHARE;
}

// h[token][f] = act(g) u from rows f and F + f of the first product, and what its rounding to bf16 dropped (lo): the second
// product takes both, which costs it 1 % and leaves y with the one rounding of the result.  g, u kept for training.
template <int ACT>
__global__ void __launch_bounds__(few::TILE * MAX_SHARE) few_gate_kernel(const float* __restrict__ part, const few::Cut cut, int F,
                                                                         __nv_bfloat16* __restrict__ h, __nv_bfloat16* __restrict__ lo,
                                                                         const Kept kept) {
  __shared__ FewSums share;
  const int col = blockIdx.x * few::TILE + threadIdx.x, f = min(col, F - 1), tok0 = blockIdx.y * TOKS;   // past the last column: repeats it
  few::wait_for_input();
  few::let_next_start();
  float s[2][TOKS];
  few_sum<2>(part, cut, {f, F + f}, tok0, &share, s);
  if (threadIdx.y > 0) return;
  const float (&g)[TOKS] = s[0], (&u)[TOKS] = s[1];
#pragma unroll
  for (int j = 0; j < TOKS; ++j) {
    const long long tok = tok0 + j;
    if (tok >= cut.tokens) break;
    if (col < F) {
      const float v = act_of<ACT>(g[j]) * u[j];
      const __nv_bfloat16 hi = __float2bfloat16(v);
      const float back = __bfloat162float(hi);
      h[tok * F + f] = hi;
      lo[tok * F + f] = __float2bfloat16(isfinite(back) ? v - back : 0.f);
    }
    if (kept.v) {                             // a warp holds a group of 32 columns
      const uint32_t gp = power_for(warp_max(gate_size<ACT>(g[j]))), up = power_for(warp_max(fabsf(u[j])));
      if (col < F) {
        const uint32_t p = saturated_half2(g[j] * power_of(gp), u[j] * power_of(up));
        kept.v[tok * 2 * F + f] = __ushort_as_half(uint16_t(p));
        kept.v[tok * 2 * F + F + f] = __ushort_as_half(uint16_t(p >> 16));
      }
      if ((threadIdx.x & 31) == 0 && col < F) {
        uint8_t* e = kept.power + (long long)(f >> 5) * cut.tokens + tok;
        e[0] = uint8_t(gp);
        e[kept.plane] = uint8_t(up);
      }
    }
  }
}

__global__ void __launch_bounds__(few::TILE * MAX_SHARE) few_sum_kernel(const float* __restrict__ part, const few::Cut cut, int N,
                                                                        __nv_bfloat16* __restrict__ y) {
  __shared__ FewSums share;
  const int col = blockIdx.x * few::TILE + threadIdx.x, n = min(col, N - 1), tok0 = blockIdx.y * TOKS;
  few::wait_for_input();
  float s[1][TOKS];
  few_sum<1>(part, cut, {n}, tok0, &share, s);
  if (threadIdx.y > 0 || col >= N) return;
#pragma unroll
  for (int j = 0; j < TOKS; ++j)
    if (tok0 + j < cut.tokens) y[(long long)(tok0 + j) * N + n] = __float2bfloat16(s[0][j]);
}

// Tokens up to which the weights are streamed by few_rows.cu.  Device time, streamed and in tiles, in us:
//   hidden x ffn    1 token       24           64          128
//   4096 x 21504    93 / 144     98 / 115    104 / 118    116 / 123
//   3584 x 18944    76 / 101     77 /  83     82 /  86     91 /  90
//   1024 x  2048    13 /  20     14 /  18     15 /  18     19 /  20
//    256 x   512    11 /  10     11 /  10     12 /  10     11 /  11
constexpr int FEW_TOKENS = few::MAX_ROWS;

// floats of the partial tiles, the larger of the two products', in whole 16 bytes; lo lies behind them
static long long few_floats(const few::Cut& a, const few::Cut& b) { return a.floats() > b.floats() ? a.floats() : b.floats(); }

static int few_forward(const void* x, long long ldx, const void* w1, const void* w2, const Kept& kept, __nv_bfloat16* h, __nv_bfloat16* y,
                       float* ws, int M, int H, int F, int Ho, int act, int* err, cudaStream_t stream) {
  const few::Cut c1 = few::cut_for(M, 2 * F, H), c2 = few::cut_for(M, Ho, F);
  __nv_bfloat16* lo = reinterpret_cast<__nv_bfloat16*>(ws + few_floats(c1, c2));
  int rc = few::launch_partials(x, nullptr, ldx, w1, ws, c1, 2 * F, H, false, err, stream);
  if (rc) return rc;
  const dim3 grid((F + few::TILE - 1) / few::TILE, (M + TOKS - 1) / TOKS), block(few::TILE, few_share(c1));
  switch (act) {
    case SILU: rc = few::launch_early(few_gate_kernel<SILU>, grid, block, 0, stream, ws, c1, F, h, lo, kept); break;
    case GELU_TANH: rc = few::launch_early(few_gate_kernel<GELU_TANH>, grid, block, 0, stream, ws, c1, F, h, lo, kept); break;
    case RELU: rc = few::launch_early(few_gate_kernel<RELU>, grid, block, 0, stream, ws, c1, F, h, lo, kept); break;
    default: rc = -10;
  }
  if (!rc) rc = few::launch_partials(h, lo, F, w2, ws, c2, Ho, F, true, err, stream);
  if (!rc) rc = few::launch_early(few_sum_kernel, dim3((Ho + few::TILE - 1) / few::TILE, (M + TOKS - 1) / TOKS), dim3(few::TILE, few_share(c2)), 0,
                                  stream, ws, c2, Ho, y);
  return rc;
}

static bool tma_ok(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

}  // namespace mlp
}  // namespace cm

using namespace cm;

// Bytes that the forward keeps for the backward beside x and h.
extern "C" long long cm_gated_mlp_kept(int M, int F) { return mlp::Kept::bytes(M, F); }

// Floats of work space that the forward needs; 0: none.
extern "C" long long cm_gated_mlp_fwd_ws(int M, int H, int F, int Ho) {
  if (M <= 0) return 0;
  if (M > mlp::FEW_TOKENS) return split::plan(sm_count(), M, Ho, F, false).floats;
  return mlp::few_floats(few::cut_for(M, 2 * F, H), few::cut_for(M, Ho, F)) + (long long)M * F / 2;
}

// y[M, Ho] = (act(x w1[:F]^T) * (x w1[F:]^T)) w2^T; x [M, H] with row pitch ldx, w1 [2F, H], w2 [Ho, F], h [M, F]; kept: cm_gated_mlp_kept
// bytes, or null.  act: 0 silu, 1 gelu (tanh form), 2 relu.  ws: cm_gated_mlp_fwd_ws floats of work space.
extern "C" int cm_gated_mlp_fwd(const void* x, long long ldx, const void* w1, const void* w2, void* kept, void* h, void* y, float* ws, int M,
                                int H, int F, int Ho, int act, int* err, cudaStream_t stream) {
  if (M <= 0 || H <= 0 || F <= 0 || Ho <= 0) return 0;
  if (H % 8 || F % 8 || Ho % 8 || !mlp::tma_ok(x, ldx) || !mlp::tma_ok(w1, H) || !mlp::tma_ok(w2, F) || !mlp::tma_ok(kept, 0) ||
      !mlp::tma_ok(h, F) || !mlp::tma_ok(y, Ho))
    return -10;
  const mlp::Kept k = kept ? mlp::Kept::at(kept, M, F) : mlp::Kept{};
  if (M <= mlp::FEW_TOKENS) {
    if (!ws) return -10;
    return mlp::few_forward(x, ldx, w1, w2, k, static_cast<__nv_bfloat16*>(h), static_cast<__nv_bfloat16*>(y), ws, M, H, F, Ho, act, err, stream);
  }
  mlp::Args args{M, F, H, mlp::plan_bn(M, F, false), k, err};
  CUtensorMap maps[5];
  int rc = make_tmap_2d_bf16(&maps[0], x, M, H, ldx, mlp::BM);
  if (!rc) rc = make_tmap_2d_bf16(&maps[1], w1, 2ll * F, H, H, args.bn / 2);
  if (!rc) rc = mlp::make_out_map(&maps[2], h, M, F, F);
  maps[3] = maps[4] = maps[2];
  if (!rc && kept) rc = mlp::make_out_map(&maps[3], k.v, M, F, 2ll * F);
  if (!rc && kept) rc = mlp::make_out_map(&maps[4], k.v + F, M, F, 2ll * F);
  if (rc) return rc;
  rc = mlp::launch_act<false>(act, maps, args, stream);
  if (rc) return rc;
  return split::gemm(h, w2, y, M, Ho, F, F, F, Ho, false, false, false, false, ws, err, stream);
}

// Floats of work space that the backward needs; 0: none.
extern "C" long long cm_gated_mlp_bwd_ws(int M, int H, int F, int Ho) {
  if (M <= 0) return 0;
  const int sms = sm_count();
  const long long n[3] = {split::plan(sms, M, H, 2 * F, true).floats, split::plan(sms, 2 * F, H, M, true).floats,
                          split::plan(sms, Ho, F, M, true).floats};
  return n[0] > n[1] ? (n[0] > n[2] ? n[0] : n[2]) : (n[1] > n[2] ? n[1] : n[2]);
}

// Gradients from dy [M, Ho] (row pitch lddy): dgu [M, 2F] is work space; dx [M, H], dw1, dw2 may be null.  dw1 / dw2: fp32 or bf16
// (dw*_fp32), added to what is there with acc*.  ws: cm_gated_mlp_bwd_ws floats of work space.
extern "C" int cm_gated_mlp_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* w1, const void* w2, const void* kept,
                                const void* h, void* dgu, void* dx, void* dw1, int dw1_fp32, int acc1, void* dw2, int dw2_fp32, int acc2,
                                float* ws, int M, int H, int F, int Ho, int act, int* err, cudaStream_t stream) {
  if (M <= 0 || H <= 0 || F <= 0 || Ho <= 0) return 0;
  if (H % 8 || F % 8 || Ho % 8 || !mlp::tma_ok(dy, lddy) || !mlp::tma_ok(x, ldx) || !mlp::tma_ok(w1, H) || !mlp::tma_ok(w2, F) ||
      !mlp::tma_ok(kept, 0) || !mlp::tma_ok(h, F) || !mlp::tma_ok(dgu, 0))
    return -10;
  int rc = 0;
  if (dx || dw1) {
    mlp::Args args{M, F, Ho, mlp::plan_bn(M, F, true), mlp::Kept::at(const_cast<void*>(kept), M, F), err};
    CUtensorMap maps[5];
    rc = make_tmap_2d_bf16(&maps[0], dy, M, Ho, lddy, mlp::BM);
    if (!rc) rc = make_tmap_2d_bf16(&maps[1], w2, Ho, F, F, 64);
    if (!rc) rc = mlp::make_out_map(&maps[3], dgu, M, F, 2ll * F);
    if (!rc) rc = mlp::make_out_map(&maps[4], static_cast<__nv_bfloat16*>(dgu) + F, M, F, 2ll * F);
    maps[2] = maps[3];
    if (!rc) rc = mlp::launch_act<true>(act, maps, args, stream);
    if (!rc && dx) rc = split::gemm(dgu, w1, dx, M, H, 2 * F, 2ll * F, H, H, false, true, false, false, ws, err, stream);
    if (!rc && dw1) rc = split::gemm(dgu, x, dw1, 2 * F, H, M, 2ll * F, ldx, H, true, true, dw1_fp32, acc1, ws, err, stream);
  }
  if (!rc && dw2) rc = split::gemm(dy, h, dw2, Ho, F, M, lddy, F, F, true, true, dw2_fp32, acc2, ws, err, stream);
  return rc;
}
