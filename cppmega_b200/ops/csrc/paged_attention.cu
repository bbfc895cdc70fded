// Attention of one new token per sequence over a paged key-value cache:
//
//   s[j] = scale * q[b, h, :] . K[j, g, :]     o[b, h, :] = sum_j softmax(s)[j] V[j, g, :]     j < lens[b], g = h / (heads of a group)
//
// where row j lies in page table[b, j / page], and an E4M3 cache holds rows divided by a power of two each.
//
// What bounds it: the cache is read once, and that is all of the time.  So every SM streams the same number of bytes without a pause:
// the keys of all sequences form one sequence of steps of 16 keys, cut into equal runs (lengths are known on the device alone, so each
// warp adds them up for itself).  A run belongs to up to 16 neighbouring warps, one per key head: they read the same tokens at the same
// time, so that memory is read in whole token rows.  A warp works alone: no barrier, its own ring of asynchronous copies (96 KB and
// more on their way per SM), its own running maximum and sum, its own accumulators.  Where a run ends inside a pair, the warp leaves its maximum,
// sum and accumulators in a work space, and a second kernel joins them in a fixed order; a pair that lies inside one run is finished at once.
//
// The products are 16 x 8 x 16 matrix instructions with 16 keys (then 16 value columns) as rows and the heads of a group as columns, eight
// at a time: S' = K q', o' = V' p'.  With the heads as rows, half of each instruction, of the exponentials and of the accumulators would belong
// to nobody at 4 to 8 heads a key.  Any order of the summed index and any order of the value columns will do as long as both factors
// agree, so a fragment is read from shared memory as the 16 bytes that lie together in a row.  A warp copies whole rows (a lane that copied its own fragments
// would ask for 16 bytes each of four rows, and every sector of V came twice), to places from which both sides of the
// exchange find their eight lanes in eight banks; the weights alone are transposed, 8 x 8 at a time.
// E4M3 becomes fp16 in one conversion per two values, exactly; the query is scaled to fp16's range by a power of two per head, the key's power
// goes into the score, and the value's power into the exponent of its weight, whose reference is a maximum of its own: weights never leave
// fp16's range, whatever the powers are.  A row of zeros has no power (its byte says 1): it sets no reference, under which the weights of the
// others would fall out of the range (a key far above the rest whose values are zero and theirs 0.05: the result was off by a quarter).
// Weights are rounded to the type of the products (bf16 or fp16: half a step of the result's own type, averaged over the keys).  Over a 16-bit cache
// the sum that divides the result is that of the rounded weights: a row that settles on few keys does not take their rounding into its result
// (1000 keys, one in fifty three times as large: off by 1.7e-3 of its norm, 2.3e-3 with the sum of the others).  Over an E4M3 cache the weights that are rounded have the
// values' powers in them, and the sum is that of the unrounded ones.  Scores, maxima, sums and accumulators are fp32.
//
// The reference value of a head's softmax follows its maximum only when that has grown by 2^8, so that accumulators are rarely rescaled.  In fp16 it
// stays 2^7 below the maximum: with weights of 1 at the most, those of keys that one key stands far above fall among the subnormals (14 above,
// its values zero: half a step is up to 4 % of such a weight).
//
// Measured, both kernels: bf16, one sequence of 131071 tokens, 64 heads over 8, 128 wide 93 us (82 at the copy rate; 64 sequences of 8192 tokens, 32
// heads over 8: 6.7 TB/s).  E4M3, 64 sequences of 100 to 16000 tokens, 32 heads over 8: 104 us (63 at the copy rate; 4.9 TB/s at 16384 each): half
// the bytes of a key, the same chain of steps, and the conversions.  Short calls are set-up (the lengths, the table, the first rows: 5 us) and the
// second kernel: 1000 tokens 9.1 us in a graph.
#include <cuda_fp16.h>

#include "few_rows.cuh"
#include "paged.cuh"

namespace cm {
namespace paged {
namespace {

constexpr int KEYS = 16;                     // keys of one step
constexpr int RING_BYTES = 192 * 1024;       // the rings of a block's warps
constexpr int SHORTEST_RUN = 2;              // steps: fewer would be all set-up, and more pieces to join
constexpr float RESCALE_AT = 8.f;            // log2
constexpr float FP16_UP = 7.f;               // log2: fp16 weights lie this far above their reference's, for more of the range below them (2^15 at most)

struct Args {
  const uint8_t* q;                          // [sequences, heads, dim]
  long long q_seq, q_head;                   // bytes
  const uint8_t *k, *v;                      // [pages, page, kv_heads, .]
  long long k_page, v_page;                  // bytes
  int k_tok, k_head, v_tok, v_head;          // bytes
  const uint8_t *k_scale, *v_scale;          // [pages, page, kv_heads] or null
  const int* table;
  long long table_row;
  const int* lens;
  void* out;                                 // [sequences, heads, vdim]
  float* part;                               // pieces of [rows][DV + 4]: weights' sum, maximum, two unused, accumulators
  int sequences, kv_heads, group, columns, pages, page, dim, vdim;
  int runs, tiles, rows;                     // runs of the sequence of steps; head tiles of a group (1, 2, 4, 8); rows of a piece
  int aligned;                               // a step lies inside one page, and its keys within 2^31 bytes
  int side, chunks;                          // key heads of a run, and how often a sequence is gone through for all of them
  float scale_log2;
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy_piece(uint32_t dst, const uint8_t* src, bool there) {
  // what is not there becomes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_whole(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pair(float lo, float hi) {
  if (BF16) return pack_bf16(lo, hi);
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF16>
__device__ __forceinline__ float2 unpair(uint32_t v) {
  if (BF16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <bool BF16>
__device__ __forceinline__ float rounded(float x) { return unpair<BF16>(pair<BF16>(x, 0.f)).x; }
// two E4M3 bytes (the lower or the upper half of a word) -> two fp16
__device__ __forceinline__ uint32_t expand_lo(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t expand_hi(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(w));
  return r;
}

__device__ __forceinline__ int length_of(const Args& a, int b, bool& bad) {
  const long long room = (long long)a.columns * a.page;
  const int n = __ldg(a.lens + b);
  if (n < 0 || n > room) bad = true;
  return n < 0 ? 0 : n > room ? (int)room : n;
}
__device__ __forceinline__ int steps_of(int len) { return (len + KEYS - 1) / KEYS; }

// steps of all (sequence, chunk of key heads) pairs, and the run length that cuts them; the same in every warp of both kernels
__device__ __forceinline__ long long all_steps(const Args& a, int lane, bool& bad) {
  long long n = 0;
  for (int b = lane; b < a.sequences; b += 32) n += steps_of(length_of(a, b, bad));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.chunks;
}
__device__ __forceinline__ long long run_length(const Args& a, long long total) {
  const long long q = (total + a.runs - 1) / a.runs;
  return q < SHORTEST_RUN ? SHORTEST_RUN : q;
}

// Warps of a block (one block per SM): as many as its registers hold, with a ring of two steps or more for each.  Per thread: 16 query
// registers and 4 DV / 16 accumulators for eight heads, and about 70 others.
__host__ __device__ constexpr int warps_of(bool e4m3, int dim, int vdim, int nt) {
  return nt == 4 ? 8 : nt == 2 ? 12 : (e4m3 ? dim + vdim : 2 * (dim + vdim)) > 384 ? 12 : 16;
}

template <bool BF16, bool E4M3, int D, int DV, int NT>
struct Form {
  static constexpr int WARPS = warps_of(E4M3, D, DV, NT);
  static constexpr bool MMA_BF16 = BF16 && !E4M3;
  static constexpr int K_ROW = E4M3 ? D : 2 * D, V_ROW = E4M3 ? DV : 2 * DV;       // bytes
  static constexpr int K_PIECES = K_ROW / 64;                 // 16-byte pieces of a key row to a lane (4 lanes a row)
  static constexpr int V_BYTES = V_ROW / 8 < 16 ? 8 : 16;     // a piece of a value row (8 lanes a row)
  static constexpr int V_PIECES = V_ROW / 8 / V_BYTES;
  static constexpr int STAGE = KEYS * (K_ROW + V_ROW);
  static constexpr int FIT = RING_BYTES / WARPS / STAGE;
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static constexpr int SPAN = V_BYTES / (E4M3 ? 1 : 2);       // neighbouring value columns of a lane's piece
  static constexpr int RING = STAGES * STAGE + (E4M3 ? STAGES * KEYS * 8 : 0);
  static_assert(STAGES >= 2 && WARPS * RING <= 227 * 1024, "a ring of two steps or more");
};

// A place in the sequence of steps
struct Place {
  int b, c, step, steps, len;                // sequence, chunk of its key heads
};
__device__ __forceinline__ void advance(const Args& a, Place& p, bool& bad) {
  if (++p.step < p.steps) return;
  p.step = 0;
  if (++p.c < a.chunks) return;
  p.c = 0;
  do {
    if (++p.b >= a.sequences) { p.steps = p.len = 0; return; }
    p.len = length_of(a, p.b, bad);
    p.steps = steps_of(p.len);
  } while (p.steps == 0);
}
// 8 x 8 values of 16 bits (row = lane / 4, two columns a lane) -> their transpose
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// over the eight lanes that hold the keys of one pair of heads
__device__ __forceinline__ float max8(float t) {
  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
  return fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
}
__device__ __forceinline__ float sum8(float t) {
  t += __shfl_xor_sync(0xffffffffu, t, 4);
  t += __shfl_xor_sync(0xffffffffu, t, 8);
  return t + __shfl_xor_sync(0xffffffffu, t, 16);
}

// BF16: type of the query and the result (fp16 otherwise; a 16-bit cache has the same); NT: tiles of eight heads that a warp multiplies
template <bool BF16, bool E4M3, int D, int DV, int NT>
__global__ void __launch_bounds__(warps_of(E4M3, D, DV, NT) * 32, 1) paged_attention_kernel(const Args a) {
  using F = Form<BF16, E4M3, D, DV, NT>;
  constexpr bool MB = F::MMA_BF16;
  constexpr float UP = MB ? 0.f : FP16_UP;
  constexpr int VT = DV / 16;                                 // 16-column tiles of the result
  extern __shared__ __align__(128) uint8_t smem_raw[];
  few::wait_for_input();                     // by every block, and before the next kernel may start: it counts on all older kernels having ended
  few::let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, row8 = lane >> 2;
  const int worker = blockIdx.x * F::WARPS + warp, lanes_of_run = a.side * a.tiles, run = worker / lanes_of_run;
  const int side = worker % lanes_of_run / a.tiles, tile = worker % a.tiles;
  const int head0 = tile * 8 * NT;                            // first head of this warp inside its group
  if (head0 >= a.group || run >= a.runs) return;
  bool bad = false;
  const long long total = all_steps(a, lane, bad), q = run_length(a, total), begin = run * q;
  const int count = (int)min(q, total - begin);               // as the shared memory, a warp's own
  if (__any_sync(0xffffffffu, bad) && a.err && lane == 0) atomicCAS(a.err, 0, ERR_BAD_ARG);
  if (begin >= total) return;

  // where the run begins
  Place at = {0, 0, 0, 0, 0};
  {
    long long before = 0;                                     // steps of the sequences before a chunk of 32
    for (int b0 = 0;; b0 += 32) {
      const int len = b0 + lane < a.sequences ? length_of(a, b0 + lane, bad) : 0;
      const long long mine = (long long)steps_of(len) * a.chunks;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > begin);
      if (past) {
        const int src = __ffs(past) - 1;
        const long long off = begin - before - __shfl_sync(0xffffffffu, upto - mine, src);
        at.len = __shfl_sync(0xffffffffu, len, src);
        at.steps = steps_of(at.len);
        at.b = b0 + src;
        at.c = (int)(off / at.steps);
        at.step = (int)(off - (long long)at.c * at.steps);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  uint8_t* ring = smem_raw + warp * F::RING;
  const uint32_t ring_s = smem_u32(ring);
  long long* rows_of = reinterpret_cast<long long*>(ring + F::STAGES * F::STAGE);      // E4M3: [stage][key] row of the scales, -1: none

  // ---- copies, STAGES - 1 steps ahead ----
  Place to = at;
  int left = count;                                           // steps not yet issued
  int col = 0, in = 0, page = -1;                             // table column, place in the page, page: of the step's first key, or of key `lane`
  auto find_page = [&]() {                                    // for a place reached by a jump
    const int pos = to.step * KEYS + (a.aligned ? 0 : lane & 15);
    col = pos / a.page;
    in = pos - col * a.page;
  };
  auto load_page = [&]() {
    page = to.step * KEYS + (a.aligned ? 0 : lane & 15) < to.len ? __ldg(a.table + to.b * a.table_row + col) : -1;
  };
  find_page();
  load_page();
  constexpr int KC = F::K_ROW / 16, VC = F::V_ROW / 16;       // 16-byte pieces of a row; 32 / KC rows to an instruction
  const int kc = lane % KC, kr = lane / KC, vc = lane % VC, vr = lane / VC;
  const bool k_exists = kc * 16 < a.dim * (E4M3 ? 1 : 2), v_exists = vc * 16 < a.vdim * (E4M3 ? 1 : 2);
  // where the copies go: K by (eight keys, piece of four lanes), V by (row of a lane's fragment, piece of eight lanes)
  const uint8_t *k_lane = a.k + kr * a.k_tok + kc * 16, *v_lane = a.v + vr * a.v_tok + vc * 16;          // aligned: within 2^31 bytes
  const uint32_t k_dst = (kc >> 2) * 512 + ((kr * 4 + (kc & 3)) ^ ((kc >> 2 & 1) * 4)) * 16;
  uint32_t v_dst[VC / 2];
#pragma unroll
  for (int i = 0; i < VC / 2; ++i) {
    const int key = i * (32 / VC) + vr, quad_of = key >> 1 & 3, y = (key & 1) | (key >> 3 << 1);
    v_dst[i] = F::V_BYTES == 16 ? ((y * F::V_PIECES + (vc >> 3)) * 32 + quad_of * 8 + ((vc & 7) ^ (2 * quad_of))) * 16
                                : y * 256 + ((vc >> 1) * 8 + quad_of * 2 + (vc & 1)) * 16;
  }
  const uint8_t *k_row = k_lane, *v_row = v_lane;             // aligned: this lane's first rows of the step
  long long scale_row = 0;                                    // and the place of its first key's exponents
  bool turned = true;                                         // the step lies in another page than the one before
  bool holes = false;                                         // pages outside the cache have been met
  auto issue = [&](int stage) {
    if (left > 0) {
      const int head = to.c * a.side + side, room = to.len - to.step * KEYS;          // key head; keys of the step
      const bool known = page >= 0 && page < a.pages;
      const uint32_t k_to = ring_s + stage * F::STAGE + k_dst, v_to = ring_s + stage * F::STAGE + KEYS * F::K_ROW;
      if (a.aligned) {
        if (!known) {
          holes = true;
          if (a.err && lane == 0) atomicCAS(a.err, 0, ERR_BAD_ARG);
        }
        const int keys = known ? room : 0;
        if (turned) {
          k_row = k_lane + page * a.k_page + (long long)in * a.k_tok + (long long)head * a.k_head;
          v_row = v_lane + page * a.v_page + (long long)in * a.v_tok + (long long)head * a.v_head;
          if (E4M3) scale_row = ((long long)page * a.page + in + lane) * a.kv_heads + head;
        } else {
          k_row += KEYS * a.k_tok;
          v_row += KEYS * a.v_tok;
          if (E4M3) scale_row += KEYS * a.kv_heads;
        }
        const uint8_t *ks = k_row, *vs = v_row;
        if (E4M3 && lane < KEYS) rows_of[stage * KEYS + lane] = lane < keys ? scale_row : -1;
        if (keys >= KEYS && a.dim == D && a.vdim == DV) {     // nothing to leave out
#pragma unroll
          for (int i = 0; i < KC / 2; ++i, ks += 32 / KC * a.k_tok)
            copy_whole(k_to + (i * (32 / KC) >> 3) * F::K_PIECES * 512 + (i * (32 / KC) & 7) * 64, ks);
#pragma unroll
          for (int i = 0; i < VC / 2; ++i, vs += 32 / VC * a.v_tok) copy_whole(v_to + v_dst[i], vs);
        } else {
#pragma unroll
          for (int i = 0; i < KC / 2; ++i, ks += 32 / KC * a.k_tok) {
            const bool there = k_exists && i * (32 / KC) + kr < keys;
            copy_piece(k_to + (i * (32 / KC) >> 3) * F::K_PIECES * 512 + (i * (32 / KC) & 7) * 64, there ? ks : a.k, there);
          }
#pragma unroll
          for (int i = 0; i < VC / 2; ++i, vs += 32 / VC * a.v_tok) {
            const bool there = v_exists && i * (32 / VC) + vr < keys;
            copy_piece(v_to + v_dst[i], there ? vs : a.v, there);
          }
        }
      } else {
        const bool there = (lane & 15) < room && known;
        const long long ko = there ? page * a.k_page + (long long)in * a.k_tok + (long long)head * a.k_head : -1;
        const long long vo = there ? page * a.v_page + (long long)in * a.v_tok + (long long)head * a.v_head : -1;
        if (!known && (lane & 15) < room && a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
        holes |= __any_sync(0xffffffffu, !known && (lane & 15) < room);
        if (E4M3 && lane < KEYS) rows_of[stage * KEYS + lane] = there ? ((long long)page * a.page + in) * a.kv_heads + head : -1;
#pragma unroll
        for (int i = 0; i < KC / 2; ++i) {
          const long long o = __shfl_sync(0xffffffffu, ko, i * (32 / KC) + kr);
          const bool here = k_exists && o >= 0;
          copy_piece(k_to + (i * (32 / KC) >> 3) * F::K_PIECES * 512 + (i * (32 / KC) & 7) * 64, here ? a.k + o + kc * 16 : a.k, here);
        }
#pragma unroll
        for (int i = 0; i < VC / 2; ++i) {
          const long long o = __shfl_sync(0xffffffffu, vo, i * (32 / VC) + vr);
          const bool here = v_exists && o >= 0;
          copy_piece(v_to + v_dst[i], here ? a.v + o + vc * 16 : a.v, here);
        }
      }
      if (--left > 0) {
        const int before = to.step;
        advance(a, to, bad);
        turned = true;
        if (to.step == before + 1 && a.page >= KEYS) {        // the next sixteen keys of the same pair
          in += KEYS;
          turned = in >= a.page;
          if (turned) {
            in -= a.page;
            ++col;
          }
        } else {
          find_page();
        }
        if (turned || !a.aligned) load_page();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // the exponents of a stage's keys (lane = key): key's power as a factor, value's power as a logarithm
  auto scales_at = [&](int stage, float& kf, float& vl) {
    kf = 1.f;
    vl = 0.f;
    if (E4M3 && lane < KEYS) {
      const long long r = rows_of[stage * KEYS + lane];
      if (r >= 0) {
        kf = power_of(__ldg(a.k_scale + r));
        vl = (float)__ldg(a.v_scale + r) - 127.f;
      }
    }
  };

#pragma unroll 1
  for (int s = 0; s < F::STAGES - 1; ++s) issue(s);
  float kf_next, vl_next;
  scales_at(0, kf_next, vl_next);

  uint32_t qf[NT][D / 16][2];                                 // query fragments: head = lane / 4
  float factor[NT][2];                                        // score factor of the heads 2 quad and 2 quad + 1, as all that follows
  float o[NT][VT][4], m[NT][2], mv[NT][2], l[NT][2];          // mv: reference of the weights that multiply V (E4M3: their own)
  const float size = fabsf(a.scale_log2);                     // the sign goes into the query, so that the largest product is the largest score
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  auto load_query = [&](const Place& p) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int head = head0 + t * 8 + row8;
      const uint8_t* src = a.q + p.b * a.q_seq + ((long long)(p.c * a.side + side) * a.group + head) * a.q_head;
      const bool row = head < a.group;
      if (!E4M3) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const int at_dim = j * 32 + quad * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row && at_dim < a.dim) v = __ldg(reinterpret_cast<const uint4*>(src + at_dim * 2));
          qf[t][2 * j][0] = v.x ^ flip;
          qf[t][2 * j][1] = v.y ^ flip;
          qf[t][2 * j + 1][0] = v.z ^ flip;
          qf[t][2 * j + 1][1] = v.w ^ flip;
        }
        factor[t][0] = factor[t][1] = size;
      } else {
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int at_dim = j * 64 + quad * 16 + c * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row && at_dim < a.dim) v = __ldg(reinterpret_cast<const uint4*>(src + at_dim * 2));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              qf[t][4 * j + 2 * c + (e >> 1)][e & 1] = w[e] ^ flip;
              const float2 f = unpair<BF16>(w[e]);
              big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // largest magnitude into [2^14, 2^15): what falls below fp16's smallest step is 2^-39 of it
        int up = 14 + 127 - (int)(__float_as_uint(big) >> 23);
        up = big > 0.f && isfinite(big) ? (up > 100 ? 100 : up < -100 ? -100 : up) : 0;
        const float by = __uint_as_float(uint32_t(127 + up) << 23);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = unpair<BF16>(qf[t][k][e]);
            qf[t][k][e] = pair<false>(f.x * by, f.y * by);
          }
        const float mine = size * __uint_as_float(uint32_t(127 - up) << 23);
        factor[t][0] = __shfl_sync(0xffffffffu, mine, quad * 8);
        factor[t][1] = __shfl_sync(0xffffffffu, mine, quad * 8 + 4);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[t][c] = mv[t][c] = -INFINITY;
        l[t][c] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < VT; ++c) o[t][c][0] = o[t][c][1] = o[t][c][2] = o[t][c][3] = 0.f;
    }
  };

  // a piece is done: the result, or what the second kernel joins
  auto leave = [&](const Place& p, int first, long long piece) {
    const bool whole = first == 0 && p.step == p.steps - 1;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float sum = sum8(l[t][c]);
        const int row = t * 8 + quad * 2 + c, head = head0 + row;
        if (head >= a.group) continue;
        float f = E4M3 && m[t][c] != -INFINITY ? ex2(mv[t][c] - m[t][c]) : 1.f;
        if (whole) {
          f = sum > 0.f ? f / sum : sum == 0.f ? 0.f : sum;   // a NaN stays
          uint8_t* dst = reinterpret_cast<uint8_t*>(a.out) + (((long long)p.b * a.kv_heads + p.c * a.side + side) * a.group + head) * a.vdim * 2;
#pragma unroll
          for (int j = 0; j < DV / 8 / F::SPAN; ++j)
#pragma unroll
            for (int e = 0; e < F::SPAN; e += 8) {
              const int column = (j * 8 + row8) * F::SPAN + e;
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int n = (j * F::SPAN + e) / 2 + i;
                w[i] = pair<BF16>(o[t][n][c] * f, o[t][n][2 + c] * f);
              }
              if (column < a.vdim) *reinterpret_cast<uint4*>(dst + column * 2) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
          float* dst = a.part + (((piece * a.side + side) * a.tiles + tile) * a.rows + row) * (DV + 4);
          if (row8 == 0) {
            dst[0] = sum;
            dst[1] = m[t][c];
          }
          dst += 4;
#pragma unroll
          for (int j = 0; j < DV / 8 / F::SPAN; ++j)
#pragma unroll
            for (int e = 0; e < F::SPAN; e += 4) {
              const int n = (j * F::SPAN + e) / 2;
              *reinterpret_cast<float4*>(dst + (j * 8 + row8) * F::SPAN + e) =
                  make_float4(o[t][n][c] * f, o[t][n][2 + c] * f, o[t][n + 1][c] * f, o[t][n + 1][2 + c] * f);
            }
        }
      }
  };

  int stage = 0, first = at.step;
  load_query(at);
  for (int i = 0; i < count; ++i) {
    copies_but<F::STAGES - 2>();
    __syncwarp();                                             // the step's rows are there, and the stage before has been read
    issue(stage == 0 ? F::STAGES - 1 : stage - 1);            // into the stage that was read last
    const float kf = kf_next, vl = vl_next;
    const int next = stage + 1 == F::STAGES ? 0 : stage + 1;
    if (E4M3 && i + 1 < count) scales_at(next, kf_next, vl_next);
    const uint32_t base = ring_s + stage * F::STAGE;

    // ---- scores: keys lane / 4 and lane / 4 + 8 of the heads 2 quad and 2 quad + 1 ----
    float s[NT][4], s2[NT][4];                                // two sums, so that a product does not wait for the one before
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[x][c] = s2[x][c] = 0.f;
#pragma unroll
    for (int j = 0; j < F::K_PIECES; ++j) {
      const uint32_t place = base + (lane ^ ((j & 1) * 4)) * 16;
      const uint4 lo = lds16(place + j * 512), hi = lds16(place + (F::K_PIECES + j) * 512);
      if (!E4M3) {
        const uint32_t k0[4] = {lo.x, hi.x, lo.y, hi.y}, k1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          mma<MB>(s[x], k0, qf[x][2 * j][0], qf[x][2 * j][1]);
          mma<MB>(s2[x], k1, qf[x][2 * j + 1][0], qf[x][2 * j + 1][1]);
        }
      } else {
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k[4] = {expand_lo(wl[e]), expand_lo(wh[e]), expand_hi(wl[e]), expand_hi(wh[e])};
#pragma unroll
          for (int x = 0; x < NT; ++x) mma<MB>(e & 1 ? s2[x] : s[x], k, qf[x][4 * j + e][0], qf[x][4 * j + e][1]);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[x][c] += s2[x][c];
    float vlog[2] = {0.f, 0.f};                               // of the two keys
    if (E4M3) {
      const float k0 = __shfl_sync(0xffffffffu, kf, row8), k1 = __shfl_sync(0xffffffffu, kf, 8 + row8);
      vlog[0] = __shfl_sync(0xffffffffu, vl, row8);
      vlog[1] = __shfl_sync(0xffffffffu, vl, 8 + row8);
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        s[x][0] *= k0; s[x][1] *= k0;
        s[x][2] *= k1; s[x][3] *= k1;
      }
    }
    const int room = at.len - at.step * KEYS;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      s[x][0] *= factor[x][0]; s[x][1] *= factor[x][1];
      s[x][2] *= factor[x][0]; s[x][3] *= factor[x][1];
    }
    if (room < KEYS) {                                        // the last step of a pair
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        if (row8 >= room) s[x][0] = s[x][1] = -INFINITY;
        if (row8 + 8 >= room) s[x][2] = s[x][3] = -INFINITY;
      }
    }
    if (holes) {                                              // those pages have no keys; nothing is kept for this case, the table is read again
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int pos = at.step * KEYS + row8 + 8 * u;
        const int p = pos < at.len ? __ldg(a.table + at.b * a.table_row + pos / a.page) : 0;
        if (p >= 0 && p < a.pages) continue;
#pragma unroll
        for (int x = 0; x < NT; ++x) s[x][2 * u] = s[x][2 * u + 1] = -INFINITY;
      }
    }

    // ---- reference values ----
    bool grown = false;
    float top[NT][2], topv[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[x][c] = fmaxf(s[x][c], s[x][2 + c]);
        grown |= top[x][c] > m[x][c] + (RESCALE_AT + UP);
        if (E4M3) {
          topv[x][c] = fmaxf(s[x][c] + vlog[0], s[x][2 + c] + vlog[1]);
          grown |= topv[x][c] > mv[x][c] + (RESCALE_AT + UP);
        }
      }
    const uint32_t vb = base + KEYS * F::K_ROW +
                        (F::V_BYTES == 16 ? (quad * 8 + (row8 ^ (2 * quad))) * 16 : ((row8 >> 2) * 8 + quad * 2 + (row8 >> 1 & 1)) * 16 + (row8 & 1) * 8);
    if (__any_sync(0xffffffffu, grown)) {
      if (E4M3) {                                             // rows of zeros: weight 0, no reference
        unsigned some = 0;                                    // a bit for each key that has values
#pragma unroll
        for (int y = 0; y < 4; ++y) {                         // keys 2 quad, + 1, + 8, + 9
          uint32_t any = 0;
#pragma unroll
          for (int j = 0; j < F::V_PIECES; ++j) {
            const uint32_t ad = vb + (y * F::V_PIECES + j) * 32 * F::V_BYTES;
            if (F::V_BYTES == 16) {
              const uint4 v = lds16(ad);
              any |= v.x | v.y | v.z | v.w;
            } else {
              const uint2 v = lds8(ad);
              any |= v.x | v.y;
            }
          }
          some |= unsigned((any & 0x7f7f7f7fu) != 0) << (2 * quad + (y & 1) + (y >> 1) * 8);
        }
        some = __reduce_or_sync(0xffffffffu, some);
        if (!(some >> row8 & 1)) vlog[0] = -INFINITY;
        if (!(some >> (row8 + 8) & 1)) vlog[1] = -INFINITY;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) topv[x][c] = fmaxf(s[x][c] + vlog[0], s[x][2 + c] + vlog[1]);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          auto raise = [&](float& ref, float t) {             // the factor that takes sums to the new reference
            t = max8(t) - UP;
            if (!(t > ref)) return 1.f;
            const float by = ex2(ref - t);
            ref = t;
            return by;
          };
          const float by = raise(m[x][c], top[x][c]);
          l[x][c] *= by;
          const float byv = E4M3 ? raise(mv[x][c], topv[x][c]) : by;
#pragma unroll
          for (int n = 0; n < VT; ++n) {
            o[x][n][c] *= byv;
            o[x][n][2 + c] *= byv;
          }
        }
    }

    // ---- weights ----
    uint32_t p[NT][2];                                        // keys 2 quad, + 1 (and + 8) of head lane / 4
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float w[4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float ref = m[x][c] == -INFINITY ? 0.f : m[x][c], refv = mv[x][c] == -INFINITY ? 0.f : mv[x][c];
        float u = ex2(s[x][c] - ref), y = ex2(s[x][2 + c] - ref);
        if (!E4M3) {                                          // the sum of what V is multiplied by
          u = rounded<MB>(u);
          y = rounded<MB>(y);
        }
        l[x][c] += u + y;
        w[c] = E4M3 ? ex2(s[x][c] + vlog[0] - refv) : u;
        w[2 + c] = E4M3 ? ex2(s[x][2 + c] + vlog[1] - refv) : y;
      }
      p[x][0] = transposed(pair<MB>(w[0], w[1]));
      p[x][1] = transposed(pair<MB>(w[2], w[3]));
    }

    // ---- values times weights ----
#pragma unroll
    for (int j = 0; j < F::V_PIECES; ++j) {
      uint32_t r[4][4];                                       // keys 2 quad, + 1, + 8, + 9
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t ad = vb + (y * F::V_PIECES + j) * 32 * F::V_BYTES;
        if (F::V_BYTES == 16) {
          const uint4 v = lds16(ad);
          r[y][0] = v.x; r[y][1] = v.y; r[y][2] = v.z; r[y][3] = v.w;
        } else {
          const uint2 v = lds8(ad);
          r[y][0] = v.x; r[y][1] = v.y; r[y][2] = r[y][3] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < F::V_BYTES / 4; ++w) {
        if (!E4M3) {
          const uint32_t v[4] = {__byte_perm(r[0][w], r[1][w], 0x5410), __byte_perm(r[0][w], r[1][w], 0x7632),
                                 __byte_perm(r[2][w], r[3][w], 0x5410), __byte_perm(r[2][w], r[3][w], 0x7632)};
#pragma unroll
          for (int x = 0; x < NT; ++x) mma<MB>(o[x][j * F::SPAN / 2 + w], v, p[x][0], p[x][1]);
        } else {
          const uint32_t e0 = __byte_perm(r[0][w], r[1][w], 0x5140), e1 = __byte_perm(r[2][w], r[3][w], 0x5140);
          const uint32_t f0 = __byte_perm(r[0][w], r[1][w], 0x7362), f1 = __byte_perm(r[2][w], r[3][w], 0x7362);
          const uint32_t v0[4] = {expand_lo(e0), expand_hi(e0), expand_lo(e1), expand_hi(e1)};
          const uint32_t v1[4] = {expand_lo(f0), expand_hi(f0), expand_lo(f1), expand_hi(f1)};
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            mma<MB>(o[x][j * F::SPAN / 2 + 2 * w], v0, p[x][0], p[x][1]);
            mma<MB>(o[x][j * F::SPAN / 2 + 2 * w + 1], v1, p[x][0], p[x][1]);
          }
        }
      }
    }

    const bool last = i + 1 == count;
    if (last || at.step == at.steps - 1) leave(at, first, run + (long long)at.b * a.chunks + at.c);
    if (!last) {
      const bool other = at.step == at.steps - 1;
      advance(a, at, bad);
      if (other) {
        first = at.step;
        load_query(at);
      }
    }
    stage = next;
  }
  copies_but<0>();
}

// The pieces of each pair become its result: a block per (sequence, head).  Piece numbers: run r leaves piece r + s of pair s, which no other
// pair of r and s shares along the sequence of steps.  All maxima are read first, so that the accumulators come without waiting for one another.
template <bool BF16, int DV, int JOIN_WARPS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const Args a, int tile_rows) {
  constexpr int C = DV / 32, AHEAD = 8;      // columns of a lane
  constexpr int JOIN_PIECES = JOIN_WARPS * 32;                // pieces weighed at once
  __shared__ float part[JOIN_WARPS][DV], weight[JOIN_PIECES], tops[JOIN_WARPS], sums[JOIN_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / (a.kv_heads * a.group), hq = blockIdx.x % (a.kv_heads * a.group), h = hq / a.group, head = hq % a.group;
  bool bad = false;
  const long long q = run_length(a, all_steps(a, lane, bad));
  long long before = 0;
  for (int i = lane; i < b; i += 32) before += steps_of(length_of(a, i, bad));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const int steps = steps_of(length_of(a, b, bad)), chunk = h / a.side;
  const long long s0 = before * a.chunks + (long long)chunk * steps;
  const int r0 = (int)(s0 / q), r1 = steps ? (int)((s0 + steps - 1) / q) : r0;
  few::wait_for_input();                     // by every block, as above
  few::let_next_start();
  if (bad && blockIdx.x == 0 && a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);   // of a table of no columns nobody else has looked at the lengths
  if (steps && r0 == r1) return;             // finished by the one run that holds it

  float top = -INFINITY, sum = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  // a piece of the next run lies `pitch` floats behind
  const long long pitch = (long long)a.side * a.tiles * a.rows * (DV + 4);
  const float* base = a.part + (long long)(b * (long long)a.chunks + chunk + r0) * pitch +
                      ((h - chunk * a.side) * a.tiles + head / tile_rows) * (long long)a.rows * (DV + 4) + (head % tile_rows) * (DV + 4);
  const int n = steps ? r1 - r0 + 1 : 0;
  for (int i0 = 0; i0 < n; i0 += JOIN_PIECES) {
    const int i = i0 + threadIdx.x, here = min(JOIN_PIECES, n - i0);
    const float ref = i < n ? base[i * pitch + 1] : -INFINITY, mass = i < n ? base[i * pitch] : 0.f;
    const float most = warp_max(ref);
    __syncthreads();                         // the weights before have been used
    if (lane == 0) tops[warp] = most;
    __syncthreads();
    float now = top;
    for (int w = 0; w < JOIN_WARPS; ++w) now = fmaxf(now, tops[w]);
    const float by = ref == -INFINITY ? 0.f : ex2(ref - now), old = top == -INFINITY ? 0.f : ex2(top - now);
    weight[threadIdx.x] = by;
    sum = sum * old + mass * by;
    top = now;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] *= old;
    __syncthreads();
    for (int k = warp; k < here; k += JOIN_WARPS * AHEAD) {
      float v[AHEAD][C], w[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int at = k + u * JOIN_WARPS;
        w[u] = at < here ? weight[at] : 0.f;
        const float* src = base + (i0 + (at < here ? at : 0)) * pitch + 4 + lane * C;
        if (C == 4) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          v[u][0] = x.x; v[u][1] = x.y; v[u][C - 2] = x.z; v[u][C - 1] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src);
          v[u][0] = x.x; v[u][1] = x.y;
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] += v[u][c] * w[u];
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
#pragma unroll
  for (int c = 0; c < C; ++c) part[warp][lane * C + c] = acc[c];
  __syncthreads();
  const int col = threadIdx.x * 2;
  if (col >= a.vdim) return;
  float mass = 0.f, x = 0.f, y = 0.f;
  for (int w = 0; w < JOIN_WARPS; ++w) {
    mass += sums[w];
    x += part[w][col];
    y += part[w][col + 1];
  }
  const float inv = mass > 0.f ? 1.f / mass : mass == 0.f ? 0.f : mass;
  reinterpret_cast<uint32_t*>(a.out)[((long long)blockIdx.x * a.vdim + col) >> 1] = pair<BF16>(x * inv, y * inv);
}

struct Layout {
  int nt, tiles, rows, grid, warps, dim, vdim, side, chunks, runs;
  long long floats;
};

// Heads of a group in tiles of eight: up to four tiles a warp with 64 value columns, two with 128 (its registers hold no more); more go to
// neighbouring warps, which read the same keys at the same time, out of L2 (32 heads on one key head of 128 and 64, 48 sequences of 32768: 121 us
// with four tiles a warp, 143 with two warps of two).
Layout layout_of(int sequences, int kv_heads, int group, int dim, int vdim, int columns, int page, bool e4m3) {
  Layout s;
  s.vdim = vdim <= 64 ? 64 : 128;
  s.dim = dim <= 64 && s.vdim == 64 ? 64 : 128;
  s.nt = group <= 8 ? 1 : group <= 16 || s.vdim == 128 ? 2 : 4;
  s.tiles = 1;
  while (s.tiles * 8 * s.nt < group) s.tiles *= 2;
  s.warps = warps_of(e4m3, s.dim, s.vdim, s.nt);
  s.rows = group < 8 * s.nt ? group : 8 * s.nt;
  s.side = kv_heads < 16 ? kv_heads : 16;                     // the largest divisor of the key heads up to 16
  while (kv_heads % s.side) --s.side;
  s.chunks = kv_heads / s.side;
  const long long steps = (long long)sequences * s.chunks * (((long long)columns * page + KEYS - 1) / KEYS);
  const long long want = (steps + SHORTEST_RUN - 1) / SHORTEST_RUN * s.tiles * s.side, sms = sm_count() > 0 ? sm_count() : 1;
  const long long blocks = (want + s.warps - 1) / s.warps;
  s.grid = int(blocks < sms ? blocks : sms);
  s.runs = s.grid * s.warps / (s.side * s.tiles);
  if (s.runs == 0) {                                          // a device of few SMs: one run all the same
    s.runs = 1;
    s.grid = steps > 0 ? (s.side * s.tiles + s.warps - 1) / s.warps : 0;
  }
  s.floats = (s.runs + (long long)sequences * s.chunks) * s.side * s.tiles * s.rows * (s.vdim + 4);
  return s;
}

template <bool BF16, bool E4M3, int D, int DV, int NT>
int start(const Args& a, int grid, cudaStream_t stream) {
  using F = Form<BF16, E4M3, D, DV, NT>;
  auto kern = paged_attention_kernel<BF16, E4M3, D, DV, NT>;
  constexpr int smem = F::WARPS * F::RING;
  if (grid > 0) {
    static PerDevice cfg;
    if (cfg.first()) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -2;
      cfg.done();
    }
    // set up while the kernel before it ends (48 sequences of 500 to 8000, 32 heads on one row, call after call: 27 us, 29 without)
    if (few::launch_early(kern, dim3(grid), dim3(F::WARPS * 32), smem, stream, a)) return -3;
  }
  // few blocks have many pieces each: 16 warps read them side by side (131071 tokens, 222 pieces,
  // both kernels: 95 us, 107 with 8 warps); many blocks have few
  const int blocks = a.sequences * a.kv_heads * a.group;
  if (blocks <= 2 * sm_count()) return few::launch_early(join_kernel<BF16, DV, 16>, dim3(blocks), dim3(512), 0, stream, a, 8 * NT);
  return few::launch_early(join_kernel<BF16, DV, 4>, dim3(blocks), dim3(128), 0, stream, a, 8 * NT);
}

template <bool BF16, bool E4M3>
int pick(const Args& a, const Layout& s, cudaStream_t stream) {
  if (s.vdim == 128) return s.nt == 1 ? start<BF16, E4M3, 128, 128, 1>(a, s.grid, stream) : start<BF16, E4M3, 128, 128, 2>(a, s.grid, stream);
  if (s.dim == 128)
    return s.nt == 1   ? start<BF16, E4M3, 128, 64, 1>(a, s.grid, stream)
           : s.nt == 2 ? start<BF16, E4M3, 128, 64, 2>(a, s.grid, stream)
                       : start<BF16, E4M3, 128, 64, 4>(a, s.grid, stream);
  return s.nt == 1   ? start<BF16, E4M3, 64, 64, 1>(a, s.grid, stream)
         : s.nt == 2 ? start<BF16, E4M3, 64, 64, 2>(a, s.grid, stream)
                     : start<BF16, E4M3, 64, 64, 4>(a, s.grid, stream);
}

}  // namespace
}  // namespace paged
}  // namespace cm

using namespace cm;
using namespace cm::paged;

extern "C" long long cm_paged_attention_ws(int sequences, int kv_heads, int group, int dim, int vdim, int columns, int page, int e4m3) {
  return layout_of(sequences, kv_heads, group, dim, vdim, columns, page, e4m3).floats;
}

// q [sequences, kv_heads * group, dim]; caches [pages, page, kv_heads, .], E4M3 ones with their exponent bytes; table [sequences, columns],
// lens [sequences]; out [sequences, kv_heads * group, vdim] packed; ws: cm_paged_attention_ws floats.  Sizes and strides (elements) come in n:
//   strides of q's sequences and heads, of pages, tokens and heads of the key cache, then of the value cache, of the table's rows;
//   sequences, kv_heads, group, columns, pages, page, dim, vdim, kind (0 bf16, 1 fp16; a 16-bit cache has the same type), e4m3.
// dim, vdim multiples of 8 (16 in an E4M3 cache) up to 128, group up to 128; steps between tokens and heads below 2^31 bytes.
extern "C" int cm_paged_attention(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, const int* table,
                                  const int* lens, void* out, float* ws, const long long* n, float scale, int* err, cudaStream_t stream) {
  const long long sequences = n[9], kv_heads = n[10], group = n[11], columns = n[12], pages = n[13], page = n[14], dim = n[15], vdim = n[16];
  const bool e4m3 = n[18];
  if (sequences <= 0 || kv_heads <= 0) return 0;
  const int step = e4m3 ? 16 : 8, es = e4m3 ? 1 : 2;
  if (group < 1 || group > 128 || dim < step || dim > 128 || dim % step || vdim < step || vdim > 128 || vdim % step || page < 1 || columns < 0 ||
      columns * page > 0x7fffffffLL - KEYS || sequences * kv_heads * group > 0x7fffffffLL)
    return -10;
  for (int i : {3, 4, 6, 7})
    if (n[i] < -(1ll << 30) || n[i] >= 1ll << 30) return -10;
  const Layout s = layout_of((int)sequences, (int)kv_heads, (int)group, (int)dim, (int)vdim, (int)columns, (int)page, e4m3);
  Args a;
  a.q = (const uint8_t*)q;
  a.q_seq = n[0] * 2; a.q_head = n[1] * 2;
  a.k = (const uint8_t*)k;
  a.v = (const uint8_t*)v;
  a.k_page = n[2] * es; a.k_tok = int(n[3] * es); a.k_head = int(n[4] * es);
  a.v_page = n[5] * es; a.v_tok = int(n[6] * es); a.v_head = int(n[7] * es);
  a.k_scale = (const uint8_t*)k_scale;
  a.v_scale = (const uint8_t*)v_scale;
  a.table = table;
  a.table_row = n[8];
  a.lens = lens;
  a.out = out;
  a.part = ws;
  a.sequences = (int)sequences;
  a.kv_heads = (int)kv_heads;
  a.group = (int)group;
  a.columns = (int)columns;
  a.pages = (int)pages;
  a.page = (int)page;
  a.dim = (int)dim;
  a.vdim = (int)vdim;
  a.runs = s.runs;
  a.side = s.side;
  a.chunks = s.chunks;
  a.aligned = page % KEYS == 0 && llabs((long long)a.k_tok) * KEYS < 1ll << 31 && llabs((long long)a.v_tok) * KEYS < 1ll << 31;
  a.tiles = s.tiles;
  a.rows = s.rows;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err;
  if (n[17] == 0) return e4m3 ? pick<true, true>(a, s, stream) : pick<true, false>(a, s, stream);
  return e4m3 ? pick<false, true>(a, s, stream) : pick<false, false>(a, s, stream);
}
