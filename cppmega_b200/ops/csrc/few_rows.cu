// Weight matrix times few rows of activations: the weights are read once, at the memory's rate, and that is all of the time.
//
// The weights are the 128-row operand A of tcgen05.mma and the activations (up to 64 rows) its N side, so that one row costs the
// tensor cores next to nothing.  What matters is that every SM streams the same number of weight bytes without a pause: the k blocks of
// all tiles form one sequence that is cut into equal runs, one per block of a grid of one block per SM (a tile per block would leave
// most SMs idle in the last wave: 336 tiles on 148 SMs are 2.3 waves), and the TMA ring holds all of shared memory (160 KB and more in
// flight per SM).  Where a run ends inside a tile the partial sums stay in fp32 in a work space; the reader adds them in a fixed order.
// 37888 x 3584 times 24 tokens: 46 us from the first block's start to the last one's end (42 at the copy rate); the last weights arrive
// between 40 and 45.  Roles as in gemm_tcgen05.cu: warp 0 TMA, warp 1 MMA, warps 2..5 partial tiles out of TMEM; every wait is bounded.
#include "few_rows.cuh"

namespace cm {
namespace few {

constexpr int BK = 64;
constexpr int THREADS = 192;
constexpr int MAX_STAGES = 12;
constexpr int A_BYTES = TILE * BK * 2;
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int SMEM_EXTRA = 256 + 1024;      // barriers, alignment

struct Args {
  Cut cut;
  int tiles, n_pad, stages, acc_cols, tmem_cols;
  float* part;
  int early, two;            // two: a second operand of the tokens' side, multiplied into the same sums
  int* err;
};

__global__ void __launch_bounds__(THREADS, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmX2,
                const Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t b_bytes = uint32_t(args.n_pad) * BK * 2, stage_bytes = A_BYTES + (args.two ? 2 : 1) * b_bytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + args.stages * stage_bytes);
  uint64_t* empty_bar = full_bar + MAX_STAGES;
  uint64_t* tmem_full = empty_bar + MAX_STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cut& cut = args.cut;
  const long long total = (long long)args.tiles * cut.nkb, begin = (long long)blockIdx.x * cut.q;
  const long long end = begin + cut.q < total ? begin + cut.q : total;

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, args.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  const bool drain = setup_barrier(args.err);
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (drain) {
    if (args.early) wait_for_input();           // what follows in the stream may not overtake the kernel before this one
    if (warp == 1) tmem_dealloc(tmem_base, args.tmem_cols);
    return;
  }

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tmW);
      tma_prefetch_desc(&tmX);
      auto weights = [&](long long kb, uint32_t stage) {                // box [128 rows, 64 k]
        const int tile = int(kb / cut.nkb), k0 = int(kb - (long long)tile * cut.nkb) * BK;
        mbar_expect_tx(&full_bar[stage], stage_bytes);
        tma_load_2d(smem + stage * stage_bytes, &tmW, &full_bar[stage], k0, tile * TILE);
      };
      auto tokens = [&](long long kb, uint32_t stage) {                 // box [n_pad rows, 64 k]
        uint8_t* sb = smem + stage * stage_bytes + A_BYTES;
        const int k0 = int(kb % cut.nkb) * BK;
        tma_load_2d(sb, &tmX, &full_bar[stage], k0, 0);
        if (args.two) tma_load_2d(sb + b_bytes, &tmX2, &full_bar[stage], k0, 0);
      };
      // behind another kernel the ring's first round of weights does not wait for the tokens; with the tokens at hand theirs go along
      // (behind 200 KB of weights a block the first tile of them arrived 4.7 us after the start)
      const long long head = begin + args.stages < end ? begin + args.stages : end;
      for (long long kb = begin; kb < head; ++kb) {
        weights(kb, uint32_t(kb - begin));
        if (!args.early) tokens(kb, uint32_t(kb - begin));
      }
      if (args.early) {
        wait_for_input();
        for (long long kb = begin; kb < head; ++kb) tokens(kb, uint32_t(kb - begin));
      }
      uint32_t stage = 0, phase = 0;                                    // the first round's release of a stage
      for (long long kb = head; kb < end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase, abort_flag, args.err, ERR_WAIT_EMPTY)) break;
        weights(kb, stage);
        tokens(kb, stage);
        if (++stage == uint32_t(args.stages)) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc_bf16(TILE, args.n_pad, false, false);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (long long kb = begin; kb < end && ok;) {
        const long long tile_end = (kb / cut.nkb + 1) * cut.nkb, stop = tile_end < end ? tile_end : end;
        ok = mbar_wait(&tmem_empty[acc], acc_phase ^ 1, abort_flag, args.err, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * args.acc_cols;
        for (bool first = true; kb < stop; ++kb, first = false) {
          ok = mbar_wait(&full_bar[stage], phase, abort_flag, args.err, ERR_WAIT_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * stage_bytes), sb = sa + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = umma_desc_sw128(sa + k * 32, 16, 1024);
            umma_f16(d, ad, umma_desc_sw128(sb + k * 32, 16, 1024), idesc, !first || k != 0);
            if (args.two) umma_f16(d, ad, umma_desc_sw128(sb + b_bytes + k * 32, 16, 1024), idesc, 1);
          }
          umma_commit(&empty_bar[stage]);
          if (++stage == uint32_t(args.stages)) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit(&tmem_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3;
    uint32_t acc = 0, acc_phase = 0;
    let_next_start();
    if (args.early) wait_for_input();           // the partial tiles go where the kernel before this one reads
    for (long long kb = begin; kb < end;) {
      const int tile = int(kb / cut.nkb);
      const long long tile_end = (long long)(tile + 1) * cut.nkb;
      kb = tile_end < end ? tile_end : end;
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, abort_flag, args.err, ERR_WAIT_TMEM_FULL))) break;
      tc_fence_after();
      float* out = args.part + cut.at(blockIdx.x, tile) + q * 32 + lane;
      const uint32_t t_base = tmem_base + acc * args.acc_cols + (uint32_t(q * 32) << 16);
      for (int c = 0; c < cut.tokens; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32(t_base + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < cut.tokens) out[(long long)(c + j) * TILE] = __uint_as_float(r[j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // let TMA copies and MMAs still in flight land before the shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, args.tmem_cols);
  }
}

Cut cut_for(int tokens, int N, int K) {
  Cut c;
  c.tokens = tokens;
  c.nkb = (K + BK - 1) / BK;
  const long long total = (long long)((N + TILE - 1) / TILE) * c.nkb, sms = sm_count() > 0 ? sm_count() : 1;
  // runs of at least 4 k blocks: a shorter one is all set-up
  long long q = (total + sms - 1) / sms;
  if (q < 4) q = 4;
  c.q = int(q);
  c.grid = total < (1ll << 31) ? int((total + q - 1) / q) : 0;
  c.maxseg = (c.q - 1) / c.nkb + 2;
  return c;
}

int launch_partials(const void* X, const void* X2, long long ldx, const void* W, float* part, const Cut& cut, int N, int K, bool early, int* err,
                    cudaStream_t stream) {
  if (cut.tokens < 1 || cut.tokens > MAX_ROWS || cut.grid < 1) return -10;
  Args a;
  a.cut = cut;
  a.tiles = (N + TILE - 1) / TILE;
  a.n_pad = (cut.tokens + 15) / 16 * 16;
  a.acc_cols = (a.n_pad + 31) / 32 * 32;        // whole 32-column reads stay inside an accumulator's columns
  a.tmem_cols = 64;
  while (a.tmem_cols < 2 * a.acc_cols) a.tmem_cols *= 2;
  a.two = X2 != nullptr;
  const int stage_bytes = A_BYTES + (a.two ? 2 : 1) * a.n_pad * BK * 2;
  a.stages = (SMEM_LIMIT - SMEM_EXTRA) / stage_bytes;
  if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
  a.part = part;
  a.early = early;
  a.err = err;
  CUtensorMap tmW, tmX, tmX2;
  int rc = make_tmap_2d_bf16(&tmW, W, N, K, K, TILE);
  if (!rc) rc = make_tmap_2d_bf16(&tmX, X, cut.tokens, K, ldx, a.n_pad);
  tmX2 = tmX;
  if (!rc && X2) rc = make_tmap_2d_bf16(&tmX2, X2, cut.tokens, K, ldx, a.n_pad);
  if (rc) return rc;
  static PerDevice configured;
  if (configured.first()) {
    if (cudaFuncSetAttribute(few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT) != cudaSuccess) return -2;
    configured.done();
  }
  const int smem = a.stages * stage_bytes + SMEM_EXTRA;
  if (early) return launch_early(few_rows_kernel, dim3(cut.grid), dim3(THREADS), smem, stream, tmW, tmX, tmX2, a);
  few_rows_kernel<<<cut.grid, THREADS, smem, stream>>>(tmW, tmX, tmX2, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace few
}  // namespace cm
