// Attention of one new token per sequence over a paged key-value cache:
//
//   s[j] = scale * q[b, h, :] . K[j, g, :]     o[b, h, :] = sum_j softmax(s)[j] V[j, g, :]     j < lens[b], g = h / (heads of a group)
//
// where row j lies in page table[b, j / page], and an E4M3 cache holds rows divided by a power of two each.
//
// What bounds it: the cache is read once, and that is all of the time.  So every SM streams the same number of bytes without a pause:
// the keys of all (sequence, key head) pairs form one sequence of steps of 16 keys, cut into equal runs, one per warp (lengths are known
// on the device alone, so each warp adds them up for itself).  A warp works alone: no barrier, its own ring of asynchronous copies (24 KB a warp,
// 192 KB an SM), its own running maximum and sum, its own accumulators.  Where a run ends inside a pair, the warp leaves its maximum, sum and
// accumulators in a work space, and a second kernel joins them in a fixed order; a pair that lies inside one run is finished at once.
//
// The products are 16 x 8 x 16 matrix instructions with the heads of a group as rows: with 4 to 16 heads a key, plain multiply-adds
// would take longer than the memory does.  Any order of the summed index and any order of the value columns will do as long as both factors agree, so a
// lane copies exactly the 16-byte pieces it needs for its fragments, in global order, and reads back only what it copied itself: no
// transposition, no swizzle, no synchronisation inside a warp.  E4M3 becomes fp16 in one conversion per two values, exactly; the query is scaled to
// fp16's range by a power of two per head, the key's power goes into the score, and the value's power into the exponent of its weight,
// whose reference is a maximum of its own: weights never leave fp16's range, whatever the powers are.
// Weights are rounded to the type of the products (bf16 or fp16: half a step of the result's own type, averaged over the keys);
// scores, maxima, sums and accumulators are fp32.
//
// The reference value of a row's softmax follows its maximum only when that has grown by 2^8, so that accumulators are rarely rescaled.
#include <cuda_fp16.h>

#include "few_rows.cuh"
#include "paged.cuh"

namespace cm {
namespace paged {
namespace {

constexpr int WARPS = 8;
constexpr int KEYS = 16;                     // keys of one step
constexpr int WARP_BYTES = 24 * 1024;        // ring of one warp
constexpr int SHORTEST_RUN = 4;              // steps: fewer would be all set-up, and more pieces to join
constexpr float RESCALE_AT = 8.f;            // log2

struct Args {
  const uint8_t* q;                          // [sequences, heads, dim]
  long long q_seq, q_head;                   // bytes
  const uint8_t *k, *v;                      // [pages, page, kv_heads, .]
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;      // bytes
  const uint8_t *k_scale, *v_scale;          // [pages, page, kv_heads] or null
  const int* table;
  long long table_row;
  const int* lens;
  void* out;                                 // [sequences, heads, vdim]
  float* part;                               // pieces of [rows][DV + 4]: weights' sum, maximum, two unused, accumulators
  int sequences, kv_heads, group, columns, pages, page, dim, vdim;
  int runs, tiles, rows;                     // runs of the sequence of steps; head tiles of a group (1, 2, 4, 8); rows of a piece
  float scale_log2;
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void copy_piece(uint32_t dst, const uint8_t* src, bool there) {
  const int n = there ? BYTES : 0;           // what is not there becomes zeros
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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

// steps of all pairs, and the run length that cuts them; the same in every warp of both kernels
__device__ __forceinline__ long long all_steps(const Args& a, int lane, bool& bad) {
  long long n = 0;
  for (int b = lane; b < a.sequences; b += 32) n += steps_of(length_of(a, b, bad));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.kv_heads;
}
__device__ __forceinline__ long long run_length(const Args& a, long long total) {
  const long long q = (total + a.runs - 1) / a.runs;
  return q < SHORTEST_RUN ? SHORTEST_RUN : q;
}

template <bool BF16, bool E4M3, int D, int DV>
struct Form {
  static constexpr bool MMA_BF16 = BF16 && !E4M3;
  static constexpr int K_ROW = E4M3 ? D : 2 * D, V_ROW = E4M3 ? DV : 2 * DV;       // bytes
  static constexpr int K_PIECES = K_ROW / 64;                 // 16-byte pieces of a key row to a lane (4 lanes a row)
  static constexpr int V_BYTES = V_ROW / 8 < 16 ? 8 : 16;     // a piece of a value row (8 lanes a row)
  static constexpr int V_PIECES = V_ROW / 8 / V_BYTES;
  static constexpr int STAGE = KEYS * (K_ROW + V_ROW);
  static constexpr int STAGES = WARP_BYTES / STAGE > 6 ? 6 : WARP_BYTES / STAGE;
  static constexpr int SPAN = V_BYTES / (E4M3 ? 1 : 2);       // neighbouring value columns of a lane's piece
  static constexpr int RING = STAGES * STAGE + (E4M3 ? STAGES * KEYS * 8 : 0);
};

// A place in the sequence of steps
struct Place {
  int b, h, step, steps, len;
};
__device__ __forceinline__ void advance(const Args& a, Place& p, bool& bad) {
  if (++p.step < p.steps) return;
  p.step = 0;
  if (++p.h < a.kv_heads) return;
  p.h = 0;
  do {
    if (++p.b >= a.sequences) { p.steps = p.len = 0; return; }
    p.len = length_of(a, p.b, bad);
    p.steps = steps_of(p.len);
  } while (p.steps == 0);
}

// BF16: type of the query and the result (fp16 otherwise; a 16-bit cache has the same); MT: 16-row tiles of heads that a warp multiplies
template <bool BF16, bool E4M3, int D, int DV, int MT>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_attention_kernel(const Args a) {
  using F = Form<BF16, E4M3, D, DV>;
  constexpr bool MB = F::MMA_BF16;
  constexpr int VT = DV / 8;                                  // 8-column tiles of the result
  extern __shared__ __align__(128) uint8_t smem_raw[];
  few::let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, row8 = lane >> 2;
  const int worker = blockIdx.x * WARPS + warp, run = worker / a.tiles, tile = worker % a.tiles;
  const int head0 = tile * 16 * MT;                           // first head of this warp inside its group
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
      const long long mine = (long long)steps_of(len) * a.kv_heads;
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
        at.h = (int)(off / at.steps);
        at.step = (int)(off - (long long)at.h * at.steps);
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
  auto page_at = [&](const Place& p) {                        // lane < 16: the page of that key
    const int pos = p.step * KEYS + lane;
    return lane < KEYS && pos < p.len ? __ldg(a.table + p.b * a.table_row + pos / a.page) : -1;
  };
  int page = page_at(to);
  auto issue = [&](int stage) {
    if (left > 0) {
      const int pos = to.step * KEYS + lane;
      long long ko = -1, vo = -1;
      if (lane < KEYS && pos < to.len) {
        if (page >= 0 && page < a.pages) {
          const int in = pos % a.page;
          ko = page * a.k_page + in * a.k_tok + to.h * a.k_head;
          vo = page * a.v_page + in * a.v_tok + to.h * a.v_head;
          if (E4M3) rows_of[stage * KEYS + lane] = ((long long)page * a.page + in) * a.kv_heads + to.h;
        } else {
          if (E4M3) rows_of[stage * KEYS + lane] = -1;
          if (a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
        }
      } else if (E4M3 && lane < KEYS) {
        rows_of[stage * KEYS + lane] = -1;
      }
      uint32_t dst = ring_s + stage * F::STAGE + lane * 16;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const long long o = __shfl_sync(0xffffffffu, ko, t * 8 + row8);
#pragma unroll
        for (int j = 0; j < F::K_PIECES; ++j, dst += 512) {
          const int byte = j * 64 + quad * 16;
          const bool there = o >= 0 && byte < a.dim * (E4M3 ? 1 : 2);
          copy_piece<16>(dst, a.k + (there ? o + byte : 0), there);
        }
      }
      dst = ring_s + stage * F::STAGE + KEYS * F::K_ROW + lane * F::V_BYTES;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long o = __shfl_sync(0xffffffffu, vo, quad * 2 + (i & 1) + (i >> 1) * 8);
#pragma unroll
        for (int j = 0; j < F::V_PIECES; ++j, dst += 32 * F::V_BYTES) {
          const int byte = j * 128 + row8 * F::V_BYTES;
          const bool there = o >= 0 && byte < a.vdim * (E4M3 ? 1 : 2);
          copy_piece<F::V_BYTES>(dst, a.v + (there ? o + byte : 0), there);
        }
      }
      --left;
      if (left > 0) {
        advance(a, to, bad);
        page = page_at(to);
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

#pragma unroll
  for (int s = 0; s < F::STAGES - 1; ++s) issue(s);
  float kf_next, vl_next;
  scales_at(0, kf_next, vl_next);

  uint32_t qf[MT][D / 16][4];                                 // query fragments
  float factor[MT][2];                                        // score factor of the rows lane / 4 and lane / 4 + 8
  float o[MT][VT][4], m[MT][2], mv[MT][2], l[MT][2];          // mv: reference of the weights that multiply V (E4M3: their own)
  auto load_query = [&](const Place& p) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int head = head0 + t * 16 + half * 8 + row8;
        const uint8_t* src = a.q + p.b * a.q_seq + ((long long)p.h * a.group + head) * a.q_head;
        const bool row = head < a.group;
        if (!E4M3) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int at_dim = j * 32 + quad * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row && at_dim < a.dim) v = __ldg(reinterpret_cast<const uint4*>(src + at_dim * 2));
            qf[t][2 * j][half] = v.x;
            qf[t][2 * j][2 + half] = v.y;
            qf[t][2 * j + 1][half] = v.z;
            qf[t][2 * j + 1][2 + half] = v.w;
          }
          factor[t][half] = a.scale_log2;
        } else {
          uint32_t raw[D / 64][8];
          float big = 0.f;
#pragma unroll
          for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int at_dim = j * 64 + quad * 16 + c * 8;
              uint4 v = make_uint4(0, 0, 0, 0);
              if (row && at_dim < a.dim) v = __ldg(reinterpret_cast<const uint4*>(src + at_dim * 2));
              raw[j][c * 4] = v.x; raw[j][c * 4 + 1] = v.y; raw[j][c * 4 + 2] = v.z; raw[j][c * 4 + 3] = v.w;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpair<BF16>(raw[j][c * 4 + e]);
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
          for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 f = unpair<BF16>(raw[j][e]);
              qf[t][4 * j + (e >> 1)][(e & 1) * 2 + half] = pair<false>(f.x * by, f.y * by);
            }
          factor[t][half] = a.scale_log2 * __uint_as_float(uint32_t(127 - up) << 23);
        }
        m[t][half] = mv[t][half] = -INFINITY;
        l[t][half] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < VT; ++c) o[t][c][0] = o[t][c][1] = o[t][c][2] = o[t][c][3] = 0.f;
    }
  };

  // a piece is done: the result, or what the second kernel joins
  auto leave = [&](const Place& p, int first, long long piece) {
    const bool whole = first == 0 && p.step == p.steps - 1;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float sum = l[t][half];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int row = t * 16 + half * 8 + row8, head = head0 + row;
        if (head >= a.group) continue;
        float f = E4M3 && m[t][half] != -INFINITY ? ex2(mv[t][half] - m[t][half]) : 1.f;
        if (whole) {
          f = sum > 0.f ? f / sum : sum == 0.f ? 0.f : sum;   // a NaN stays
          uint8_t* dst = reinterpret_cast<uint8_t*>(a.out) + (((long long)p.b * a.kv_heads + p.h) * a.group + head) * a.vdim * 2;
#pragma unroll
          for (int j = 0; j < VT / F::SPAN; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < F::SPAN; e += 8) {
                const int col = (j * 8 + quad * 2 + c) * F::SPAN + e;
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = pair<BF16>(o[t][j * F::SPAN + e + 2 * i][half * 2 + c] * f, o[t][j * F::SPAN + e + 2 * i + 1][half * 2 + c] * f);
                if (col < a.vdim) *reinterpret_cast<uint4*>(dst + col * 2) = make_uint4(w[0], w[1], w[2], w[3]);
              }
        } else {
          float* dst = a.part + ((piece * a.tiles + tile) * a.rows + row) * (DV + 4);
          if (quad == 0) {
            dst[0] = sum;
            dst[1] = m[t][half];
          }
          dst += 4;
#pragma unroll
          for (int j = 0; j < VT / F::SPAN; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < F::SPAN; e += 4) {
                const int col = (j * 8 + quad * 2 + c) * F::SPAN + e, n = j * F::SPAN + e, k = half * 2 + c;
                *reinterpret_cast<float4*>(dst + col) = make_float4(o[t][n][k] * f, o[t][n + 1][k] * f, o[t][n + 2][k] * f, o[t][n + 3][k] * f);
              }
        }
      }
  };

  int stage = 0, first = at.step;
  load_query(at);
  for (int i = 0; i < count; ++i) {
    copies_but<F::STAGES - 2>();
    issue(stage == 0 ? F::STAGES - 1 : stage - 1);            // into the stage that was read last
    const float kf = kf_next, vl = vl_next;
    const int next = stage + 1 == F::STAGES ? 0 : stage + 1;
    if (E4M3 && i + 1 < count) scales_at(next, kf_next, vl_next);
    const uint32_t base = ring_s + stage * F::STAGE;

    // ---- scores ----
    float s[MT][2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int x = 0; x < MT; ++x) s[x][t][0] = s[x][t][1] = s[x][t][2] = s[x][t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < F::K_PIECES; ++j) {
        const uint4 kv = lds16(base + (t * F::K_PIECES + j) * 512 + lane * 16);
        if (!E4M3) {
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            mma<MB>(s[x][t], qf[x][2 * j], kv.x, kv.y);
            mma<MB>(s[x][t], qf[x][2 * j + 1], kv.z, kv.w);
          }
        } else {
          const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t lo = expand_lo(w[e]), hi = expand_hi(w[e]);
#pragma unroll
            for (int x = 0; x < MT; ++x) mma<MB>(s[x][t], qf[x][4 * j + e], lo, hi);
          }
        }
      }
    }
    const int room = at.len - at.step * KEYS - quad * 2;      // keys of this lane: quad * 2 + {0, 1}, + 8
    float vlog[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float kp = E4M3 ? __shfl_sync(0xffffffffu, kf, t * 8 + quad * 2 + c) : 1.f;
        vlog[t][c] = E4M3 ? __shfl_sync(0xffffffffu, vl, t * 8 + quad * 2 + c) : 0.f;
        const bool there = t * 8 + c < room;
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          s[x][t][c] = there ? s[x][t][c] * factor[x][0] * kp : -INFINITY;
          s[x][t][2 + c] = there ? s[x][t][2 + c] * factor[x][1] * kp : -INFINITY;
        }
      }

    // ---- reference values ----
    bool grown = false;
    float top[MT][2], topv[MT][2];
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = half * 2;
        top[x][half] = fmaxf(fmaxf(s[x][0][k], s[x][0][k + 1]), fmaxf(s[x][1][k], s[x][1][k + 1]));
        grown |= top[x][half] > m[x][half] + RESCALE_AT;
        if (E4M3) {
          topv[x][half] = fmaxf(fmaxf(s[x][0][k] + vlog[0][0], s[x][0][k + 1] + vlog[0][1]),
                                fmaxf(s[x][1][k] + vlog[1][0], s[x][1][k + 1] + vlog[1][1]));
          grown |= topv[x][half] > mv[x][half] + RESCALE_AT;
        }
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          auto raise = [&](float& ref, float t) {             // the factor that takes sums to the new reference
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            if (!(t > ref)) return 1.f;
            const float by = ex2(ref - t);
            ref = t;
            return by;
          };
          const float by = raise(m[x][half], top[x][half]);
          l[x][half] *= by;
          const float byv = E4M3 ? raise(mv[x][half], topv[x][half]) : by;
#pragma unroll
          for (int c = 0; c < VT; ++c) {
            o[x][c][half * 2] *= byv;
            o[x][c][half * 2 + 1] *= byv;
          }
        }
    }

    // ---- weights ----
    uint32_t p[MT][4];
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float ref = m[x][half] == -INFINITY ? 0.f : m[x][half];
        const float refv = mv[x][half] == -INFINITY ? 0.f : mv[x][half];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float u = s[x][t][half * 2], w = s[x][t][half * 2 + 1];
          const float pu = ex2(u - ref), pw = ex2(w - ref);
          l[x][half] += pu + pw;
          p[x][t * 2 + half] = E4M3 ? pair<MB>(ex2(u + vlog[t][0] - refv), ex2(w + vlog[t][1] - refv)) : pair<MB>(pu, pw);
        }
      }

    // ---- weights times values ----
    const uint32_t vb = base + KEYS * F::K_ROW + lane * F::V_BYTES;
#pragma unroll
    for (int j = 0; j < F::V_PIECES; ++j) {
      uint32_t r[4][4];
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
          const uint32_t b0 = __byte_perm(r[0][w], r[1][w], 0x5410), b1 = __byte_perm(r[2][w], r[3][w], 0x5410);
          const uint32_t c0 = __byte_perm(r[0][w], r[1][w], 0x7632), c1 = __byte_perm(r[2][w], r[3][w], 0x7632);
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            mma<MB>(o[x][j * F::SPAN + 2 * w], p[x], b0, b1);
            mma<MB>(o[x][j * F::SPAN + 2 * w + 1], p[x], c0, c1);
          }
        } else {
          const uint32_t e0 = __byte_perm(r[0][w], r[1][w], 0x5140), e1 = __byte_perm(r[2][w], r[3][w], 0x5140);
          const uint32_t f0 = __byte_perm(r[0][w], r[1][w], 0x7362), f1 = __byte_perm(r[2][w], r[3][w], 0x7362);
          const uint32_t b[4][2] = {{expand_lo(e0), expand_lo(e1)}, {expand_hi(e0), expand_hi(e1)},
                                    {expand_lo(f0), expand_lo(f1)}, {expand_hi(f0), expand_hi(f1)}};
#pragma unroll
          for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int c = 0; c < 4; ++c) mma<MB>(o[x][j * F::SPAN + 4 * w + c], p[x], b[c][0], b[c][1]);
        }
      }
    }

    const bool last = i + 1 == count;
    if (last || at.step == at.steps - 1) leave(at, first, run + (long long)at.b * a.kv_heads + at.h);
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

constexpr int JOIN_WARPS = 4;

// The pieces of each pair become its result: a block per (sequence, head).  Piece numbers: run r leaves piece r + s of pair s, which no other
// pair of r and s shares along the sequence of steps.
template <bool BF16, int DV>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const Args a, int tile_rows) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / (a.kv_heads * a.group), hq = blockIdx.x % (a.kv_heads * a.group), h = hq / a.group, head = hq % a.group;
  bool bad = false;
  const long long q = run_length(a, all_steps(a, lane, bad));
  long long before = 0;
  for (int i = lane; i < b; i += 32) before += steps_of(length_of(a, i, bad));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const int steps = steps_of(length_of(a, b, bad));
  const long long s0 = before * a.kv_heads + (long long)h * steps;
  const int r0 = (int)(s0 / q), r1 = steps ? (int)((s0 + steps - 1) / q) : r0;
  few::wait_for_input();                     // by every block: the next kernel of the stream counts on this one having waited
  if (steps && r0 == r1) return;             // finished by the one run that holds it

  constexpr int C = DV / 32;                 // columns of a lane
  __shared__ float part[JOIN_WARPS][DV + 2];
  float top = -INFINITY, sum = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  if (steps) {
    const int tile = head / tile_rows, row = head % tile_rows;
    const long long pair_no = (long long)b * a.kv_heads + h;
    for (int r = r0 + warp; r <= r1; r += JOIN_WARPS) {
      const float* src = a.part + (((r + pair_no) * a.tiles + tile) * a.rows + row) * (DV + 4);
      const float n = src[0], ref = src[1];
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = src[4 + lane * C + c];
      const float t = fmaxf(top, ref);
      const float old = top == -INFINITY ? 0.f : ex2(top - t), by = ref == -INFINITY ? 0.f : ex2(ref - t);
      sum = sum * old + n * by;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = acc[c] * old + v[c] * by;
      top = t;
    }
  }
  if (lane == 0) {
    part[warp][DV] = sum;
    part[warp][DV + 1] = top;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) part[warp][lane * C + c] = acc[c];
  __syncthreads();
  const int col = threadIdx.x * 2;
  if (col >= a.vdim) return;
  top = -INFINITY;
  for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, part[w][DV + 1]);
  float n = 0.f, x = 0.f, y = 0.f;
  for (int w = 0; w < JOIN_WARPS; ++w) {
    const float by = part[w][DV + 1] == -INFINITY ? 0.f : ex2(part[w][DV + 1] - top);
    n += part[w][DV] * by;
    x += part[w][col] * by;
    y += part[w][col + 1] * by;
  }
  const float inv = n > 0.f ? 1.f / n : n == 0.f ? 0.f : n;
  reinterpret_cast<uint32_t*>(a.out)[((long long)blockIdx.x * a.vdim + col) >> 1] = pair<BF16>(x * inv, y * inv);
}

struct Layout {
  int mt, tiles, rows, grid, dv;
  long long floats;
};

// Heads of a group in tiles of 16 rows: two tiles a warp where the accumulators leave registers for them (64 value columns), else one; more
// tiles than that go to neighbouring warps, which read the same keys at the same time, out of L2.
Layout layout_of(int sequences, int kv_heads, int group, int dim, int vdim, int columns, int page) {
  Layout s;
  s.dv = vdim <= 64 && (dim <= 128) ? 64 : 128;
  s.mt = s.dv == 64 && group > 16 ? 2 : 1;
  s.tiles = 1;
  while (s.tiles * 16 * s.mt < group) s.tiles *= 2;
  s.rows = group < 16 * s.mt ? group : 16 * s.mt;
  const long long steps = (long long)sequences * kv_heads * (((long long)columns * page + KEYS - 1) / KEYS);
  const long long want = (steps + SHORTEST_RUN - 1) / SHORTEST_RUN * s.tiles, sms = sm_count() > 0 ? sm_count() : 1;
  const long long blocks = (want + WARPS - 1) / WARPS;
  s.grid = int(blocks < sms ? blocks : sms);
  s.floats = (s.grid * WARPS / s.tiles + (long long)sequences * kv_heads) * s.tiles * s.rows * (s.dv + 4);
  return s;
}

template <bool BF16, bool E4M3, int D, int DV, int MT>
int start(const Args& a, int grid, cudaStream_t stream) {
  auto kern = paged_attention_kernel<BF16, E4M3, D, DV, MT>;
  constexpr int smem = WARPS * Form<BF16, E4M3, D, DV>::RING;
  if (grid > 0) {
    static PerDevice cfg;
    if (cfg.first()) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -2;
      cfg.done();
    }
    kern<<<grid, WARPS * 32, smem, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return -3;
  }
  const dim3 blocks((unsigned)(a.sequences * a.kv_heads * a.group));
  return few::launch_early(join_kernel<BF16, DV>, blocks, dim3(JOIN_WARPS * 32), 0, stream, a, 16 * MT);
}

template <bool BF16, bool E4M3>
int pick(const Args& a, const Layout& s, cudaStream_t stream) {
  if (s.dv == 64) {
    if (a.dim <= 64) return s.mt == 2 ? start<BF16, E4M3, 64, 64, 2>(a, s.grid, stream) : start<BF16, E4M3, 64, 64, 1>(a, s.grid, stream);
    return s.mt == 2 ? start<BF16, E4M3, 128, 64, 2>(a, s.grid, stream) : start<BF16, E4M3, 128, 64, 1>(a, s.grid, stream);
  }
  return start<BF16, E4M3, 128, 128, 1>(a, s.grid, stream);
}

}  // namespace
}  // namespace paged
}  // namespace cm

using namespace cm;
using namespace cm::paged;

extern "C" long long cm_paged_attention_ws(int sequences, int kv_heads, int group, int dim, int vdim, int columns, int page) {
  return layout_of(sequences, kv_heads, group, dim, vdim, columns, page).floats;
}

// q [sequences, kv_heads * group, dim]; caches [pages, page, kv_heads, .], E4M3 ones with their exponent bytes; table [sequences, columns],
// lens [sequences]; out [sequences, kv_heads * group, vdim] packed; ws: cm_paged_attention_ws floats.  Sizes and strides (elements) come in n:
//   strides of q's sequences and heads, of pages, tokens and heads of the key cache, then of the value cache, of the table's rows;
//   sequences, kv_heads, group, columns, pages, page, dim, vdim, kind (0 bf16, 1 fp16; a 16-bit cache has the same type), e4m3.
// dim, vdim multiples of 8 (16 in an E4M3 cache) up to 128, group up to 128.
extern "C" int cm_paged_attention(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, const int* table,
                                  const int* lens, void* out, float* ws, const long long* n, float scale, int* err, cudaStream_t stream) {
  const long long sequences = n[9], kv_heads = n[10], group = n[11], columns = n[12], pages = n[13], page = n[14], dim = n[15], vdim = n[16];
  const bool e4m3 = n[18];
  if (sequences <= 0 || kv_heads <= 0) return 0;
  const int step = e4m3 ? 16 : 8, es = e4m3 ? 1 : 2;
  if (group < 1 || group > 128 || dim < step || dim > 128 || dim % step || vdim < step || vdim > 128 || vdim % step || page < 1 || columns < 0 ||
      columns * page > 0x7fffffffLL - KEYS || sequences * kv_heads * group > 0x7fffffffLL)
    return -10;
  const Layout s = layout_of((int)sequences, (int)kv_heads, (int)group, (int)dim, (int)vdim, (int)columns, (int)page);
  Args a;
  a.q = (const uint8_t*)q;
  a.q_seq = n[0] * 2; a.q_head = n[1] * 2;
  a.k = (const uint8_t*)k;
  a.v = (const uint8_t*)v;
  a.k_page = n[2] * es; a.k_tok = n[3] * es; a.k_head = n[4] * es;
  a.v_page = n[5] * es; a.v_tok = n[6] * es; a.v_head = n[7] * es;
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
  a.runs = s.grid > 0 ? s.grid * WARPS / s.tiles : 1;
  a.tiles = s.tiles;
  a.rows = s.rows;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err;
  if (n[17] == 0) return e4m3 ? pick<true, true>(a, s, stream) : pick<true, false>(a, s, stream);
  return e4m3 ? pick<false, true>(a, s, stream) : pick<false, false>(a, s, stream);
}
