// Dense bf16 product whose last tiles share their reduction.
//
// A product of t tiles on p CTA pairs takes ceil(t / p) waves, however little the last wave has to do: 4095 x 3584 x 18944 is 224 tiles
// for 74 pairs, and its fourth wave works on two of them; a product of few tiles (a short batch, a narrow layer) leaves most pairs idle
// from the start.  Here whole waves go to cm_gemm_bf16 as they are, and the rows that are left over are computed by every pair: their
// tiles are cut along the reduction, each run leaves an fp32 partial result, and a second kernel adds the runs in a fixed order,
// rounds once, and adds to C where that is asked for.
// The kernel is the 256 x 256 x 64 tcgen05.mma.cta_group::2 pipeline of gemm_pair.cu with runs instead of whole reductions, 5 stages,
// eight epilogue warps (a pair has about one tile, so that its epilogue hides under nothing), and fp32 tiles out by bulk stores.
#include "gemm_split.cuh"
#include "pair_issue.cuh"

extern "C" int cm_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc,
                            int a_mn, int b_mn, int out_fp32, int accumulate, int* err, cudaStream_t stream);

namespace cm {
namespace split {

using namespace pair2;

constexpr int BM = 128, BK = 64, UMMA_K = 16;
constexpr int EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr int STAGES = 5;
constexpr int A_BYTES = BM * BK * 2, STAGE_BYTES = 2 * A_BYTES;
constexpr int STORE_BYTES = 32 * 128, STORE_BUFS = 2;      // a warp's 32 rows x 32 columns of fp32
constexpr int STORE_OFF = STAGES * STAGE_BYTES;
constexpr int BAR_OFF = STORE_OFF + EPI_WARPS * STORE_BUFS * STORE_BYTES;
constexpr int SMEM_TOTAL = BAR_OFF + 256 + 1024;

struct Args {
  int M, N, K, bn, slices, kb_per_slice;
  int* err;
};

template <bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmP,
             const Args args) {
  extern __shared__ uint8_t smem_raw[];
  // the dynamic segment starts at the same offset in both CTAs, so the aligned offsets agree as the descriptors need
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + BAR_OFF);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int half = args.bn >> 1;
  const int tiles_n = (args.N + args.bn - 1) / args.bn, tiles = tiles_n * ((args.M + 2 * BM - 1) / (2 * BM)), total = tiles * args.slices;
  const int nkb = (args.K + BK - 1) / BK;
  const int first_unit = blockIdx.x >> 1, unit_step = gridDim.x >> 1;
  // neighbouring pairs work on the same run of the reduction, tile after tile
  auto place = [&](int unit, int& slice, int& m0, int& n0, int& kb0, int& kb1) {
    slice = unit / tiles;
    const int t = unit - slice * tiles;
    m0 = t / tiles_n * 2 * BM;
    n0 = t % tiles_n * args.bn;
    kb0 = slice * args.kb_per_slice;
    kb1 = min(nkb, kb0 + args.kb_per_slice);
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
      for (int unit = first_unit; unit < total && ok; unit += unit_step) {
        int slice, m0, n0, kb0, kb1;
        place(unit, slice, m0, n0, kb0, kb1);
        const int ma = m0 + rank * BM, nb = n0 + rank * half;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, args.err, ERR_WAIT_EMPTY);
          if (!ok) break;
          uint8_t* sa = smem + stage * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          if (rank == 0) mbar_expect_tx(&full_bar[stage], pair_bytes);
          const uint32_t bar = map_to_rank(smem_u32(&full_bar[stage]), 0);
          const int k0 = kb * BK;
          if (!A_MN) {
            load_2d(sa, &tmA, bar, k0, ma);                                              // box [128 rows, 64 k]
          } else {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) load_2d(sa + c * (BK * 128), &tmA, bar, ma + c * 64, k0);   // boxes [64 k, 64 m]
          }
          if (!B_MN) {
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
      const uint32_t idesc = umma_idesc_bf16(2 * BM, args.bn, A_MN, B_MN);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = *abort_flag == 0;
      for (int unit = first_unit; unit < total && ok; unit += unit_step) {
        int slice, m0, n0, kb0, kb1;
        place(unit, slice, m0, n0, kb0, kb1);
        ok = mbar_wait(&tmem_empty[acc], acc_phase ^ 1, abort_flag, args.err, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, abort_flag, args.err, ERR_WAIT_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
          const uint32_t sb = sa + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t ad = A_MN ? umma_desc_sw128(sa + k * (UMMA_K * 128), BK * 128, 1024) : umma_desc_sw128(sa + k * (UMMA_K * 2), 16, 1024);
            const uint64_t bd = B_MN ? umma_desc_sw128(sb + k * (UMMA_K * 128), BK * 128, 1024) : umma_desc_sw128(sb + k * (UMMA_K * 2), 16, 1024);
            mma_2cta(d_tmem, ad, bd, idesc, kb != kb0 || k != 0);
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
    const int c_begin = ((warp - 2) >> 2) * half, c_end = c_begin + half;
    uint8_t* staging = smem + STORE_OFF + (warp - 2) * STORE_BUFS * STORE_BYTES;
    uint32_t acc = 0, acc_phase = 0, buf = 0;
    bool ok = *abort_flag == 0;
    for (int unit = first_unit; unit < total && ok; unit += unit_step) {
      int slice, m0, n0, kb0, kb1;
      place(unit, slice, m0, n0, kb0, kb1);
      const int row0 = m0 + rank * BM + q * 32;
      ok = __all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, abort_flag, args.err, ERR_WAIT_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_base = tmem_base + acc * 256 + (uint32_t(q * 32) << 16);
      if (row0 < args.M) {
        for (int c = c_begin; c < c_end && n0 + c < args.N; c += 32) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(STORE_BUFS - 1) : "memory");   // this buffer has been read
          __syncwarp();
          uint8_t* dst = staging + buf * STORE_BYTES;
          uint32_t r[32];
          tmem_ld_32x32(t_base + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<uint4*>(dst + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            bulk_store_3d(&tmP, dst, n0 + c, row0, slice);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          buf ^= 1;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&tmem_empty[acc]), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
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

// C[m][n] (+)= sum over slices of part[s][m][n]; n in groups of 4 (N % 8 == 0), rows of C with their own pitch.
template <typename T, bool ACC>
__global__ void __launch_bounds__(256) split_sum_kernel(const float4* __restrict__ part, T* __restrict__ C, long long quads, int quads_per_row,
                                                        long long ldc, int slices, int aligned) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= quads) return;
  const long long row = i / quads_per_row;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < slices; ++k) {
    const float4 v = part[k * quads + i];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  T* dst = C + row * ldc + (i - row * quads_per_row) * 4;
  const float f[4] = {s.x, s.y, s.z, s.w};
  struct alignas(4 * sizeof(T)) Quad {
    T v[4];
  } o;
  if (aligned) {
    if (ACC) o = *reinterpret_cast<const Quad*>(dst);
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = T(ACC ? float(o.v[j]) + f[j] : f[j]);
    *reinterpret_cast<Quad*>(dst) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = T(ACC ? float(dst[j]) + f[j] : f[j]);
  }
}

template <bool A_MN, bool B_MN>
static int launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmP, const Args& args, int units, cudaStream_t stream) {
  auto kern = split_kernel<A_MN, B_MN>;
  static PerDevice configured;
  if (configured.first()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_TOTAL) != cudaSuccess) return -2;
    configured.done();
  }
  const int pairs = sm_count() / 2;
  kern<<<2 * (units < pairs ? units : pairs), THREADS, SMEM_TOTAL, stream>>>(tmA, tmB, tmP, args);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// Times in us, by the tile shapes' time for a 64-deep k block (the weights of plan_dense, at 0.39 us for a 256-column pair tile) and 3 us
// of set-up and epilogue a wave; a split pays 5 us for its second kernel and the fp32 partial results at 4 TB/s.
static double unsplit_time(int sms, int M, int N, int K, bool b_mn) {
  const double nkb = (K + BK - 1) / BK;
  double best = 1e30;
  auto consider = [&](int rows, int bn, double slots, double kb) {
    const double tiles = double((M + rows - 1) / rows) * ((N + bn - 1) / bn), waves = double((long long)((tiles + slots - 1) / slots));
    const double t = waves * (kb * nkb + 3.0);
    if (t < best) best = t;
  };
  consider(256, 256, sms / 2, 0.39);
  if (!b_mn) consider(256, 192, sms / 2, 0.33);
  consider(256, 128, sms / 2, 0.287);
  consider(128, 256, sms, 0.46);
  consider(128, 128, sms, 0.289);
  consider(128, 64, sms, 0.239);
  return best;
}

Plan plan(int sms, int M, int N, int K, bool b_mn) {
  Plan none{M, 256, 0, 0, 0};
  const int pairs = sms / 2, nkb = (K + BK - 1) / BK, tm = (M + 255) / 256;
  if (pairs < 1 || nkb < 8) return none;
  double best = unsplit_time(sms, M, N, K, b_mn) * 0.95;           // a split has to be worth it
  Plan p = none;
  auto consider = [&](int whole_tiles, int bn) {              // row tiles done whole
    const int rest = M - whole_tiles * 256;
    if (rest <= 0) return;
    const int units = ((rest + 255) / 256) * ((N + bn - 1) / bn);
    int slices = pairs / units;
    if (slices > nkb / 4) slices = nkb / 4;
    if (slices > 32) slices = 32;
    if (slices < 2) return;
    const int per = (nkb + slices - 1) / slices;
    slices = (nkb + per - 1) / per;
    const double bytes = 8.0 * slices * rest * N;
    const double t = (whole_tiles ? unsplit_time(sms, whole_tiles * 256, N, K, b_mn) : 0.0) + per * (bn == 256 ? 0.39 : 0.287) + 3.0 + 5.0 + bytes / 4e6;
    if (t < best) {
      best = t;
      p = Plan{whole_tiles * 256, bn, slices, per, (long long)slices * rest * N};
    }
  };
  for (int bn = 256; bn >= 128; bn -= 128) {
    const int tn = (N + bn - 1) / bn;
    consider(0, bn);
    const int waves = int((long long)tm * ((N + 255) / 256) / pairs);       // whole waves of 256-column tiles
    const int rows = int((long long)waves * pairs / ((N + 255) / 256));
    if (waves > 0 && rows > 0 && rows < tm && (tm - rows) * tn * 2 <= pairs) consider(rows, bn);
  }
  return p;
}

static int make_part_map(CUtensorMap* out, float* part, int M, int N, int slices) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return -1;
  cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)slices};
  cuuint64_t strides[2] = {(cuuint64_t)N * 4, (cuuint64_t)N * M * 4};
  cuuint32_t box[3] = {32, 32, 1}, one[3] = {1, 1, 1};
  CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, part, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int gemm(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc, bool a_mn, bool b_mn,
         bool out_fp32, bool accumulate, float* ws, int* err, cudaStream_t stream) {
  const Plan p = plan(sm_count(), M, N, K, b_mn);
  if (!p.slices) return cm_gemm_bf16(A, B, C, M, N, K, lda, ldb, ldc, a_mn, b_mn, out_fp32, accumulate, err, stream);
  if (!ws || N % 8) return -10;
  int rc = p.whole ? cm_gemm_bf16(A, B, C, p.whole, N, K, lda, ldb, ldc, a_mn, b_mn, out_fp32, accumulate, err, stream) : 0;
  if (rc) return rc;
  const int rest = M - p.whole;
  const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(A) + (a_mn ? (long long)p.whole : p.whole * lda);
  CUtensorMap tmA, tmB, tmP;
  rc = a_mn ? make_tmap_2d_bf16(&tmA, a, K, rest, lda, 64) : make_tmap_2d_bf16(&tmA, a, rest, K, lda, BM);
  if (!rc) rc = b_mn ? make_tmap_2d_bf16(&tmB, B, K, N, ldb, 64) : make_tmap_2d_bf16(&tmB, B, N, K, ldb, p.bn / 2);
  if (!rc) rc = make_part_map(&tmP, ws, rest, N, p.slices);
  if (rc) return rc;
  const Args args{rest, N, K, p.bn, p.slices, p.kb_per_slice, err};
  const int units = ((rest + 255) / 256) * ((N + p.bn - 1) / p.bn) * p.slices;
  if (a_mn) rc = b_mn ? launch<true, true>(tmA, tmB, tmP, args, units, stream) : launch<true, false>(tmA, tmB, tmP, args, units, stream);
  else rc = b_mn ? launch<false, true>(tmA, tmB, tmP, args, units, stream) : launch<false, false>(tmA, tmB, tmP, args, units, stream);
  if (rc) return rc;
  const long long quads = (long long)rest * (N / 4);
  const unsigned grid = unsigned((quads + 255) / 256);
  const float4* part = reinterpret_cast<const float4*>(ws);
  const int aligned = ((reinterpret_cast<uintptr_t>(C) | (ldc * (out_fp32 ? 4 : 2))) & (out_fp32 ? 15 : 7)) == 0;
  if (out_fp32) {
    float* c = static_cast<float*>(C) + p.whole * ldc;
    if (accumulate) split_sum_kernel<float, true><<<grid, 256, 0, stream>>>(part, c, quads, N / 4, ldc, p.slices, aligned);
    else split_sum_kernel<float, false><<<grid, 256, 0, stream>>>(part, c, quads, N / 4, ldc, p.slices, aligned);
  } else {
    __nv_bfloat16* c = static_cast<__nv_bfloat16*>(C) + p.whole * ldc;
    if (accumulate) split_sum_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(part, c, quads, N / 4, ldc, p.slices, aligned);
    else split_sum_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(part, c, quads, N / 4, ldc, p.slices, aligned);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace split
}  // namespace cm

// The plan on a chip of `sms` SMs: out = {rows done whole, columns of a tile, slices, k blocks per slice}; returns the floats of work space.
extern "C" long long cm_gemm_split_plan(int sms, int M, int N, int K, int b_mn, int* out) {
  const cm::split::Plan p = cm::split::plan(sms, M, N, K, b_mn != 0);
  out[0] = p.whole; out[1] = p.bn; out[2] = p.slices; out[3] = p.kb_per_slice;
  return p.floats;
}

// The product with its plan on this chip; ws: the plan's floats.
extern "C" int cm_gemm_split(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc, int a_mn,
                             int b_mn, int out_fp32, int accumulate, float* ws, int* err, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return cm::split::gemm(A, B, C, M, N, K, lda, ldb, ldc, a_mn != 0, b_mn != 0, out_fp32 != 0, accumulate != 0, ws, err, stream);
}
