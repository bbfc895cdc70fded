// Causal attention over sequences of different lengths packed into one buffer, with grouped heads; forward and backward on tcgen05 with the
// scores in TMEM.
//
//   s[i, j] = scale * q[i] . k[j]   (j <= i + Lk - L inside the sequence)     p = softmax_j(s)     o[i] = sum_j p[i, j] v[j]
//   delta[i] = do[i] . o[i]    ds = p (do v' - delta)    dq = scale ds k    dk = scale ds' q    dv = p' do
//
// Rows.  A query tile is 128 rows of (token, head of a group), so one tile of keys serves all heads of a group, a short sequence fills a
// tile with its heads, the key gradients of a group add up inside one accumulator, and the tile of a causal diagonal is 128 / heads tokens
// high.  Groups that do not divide 128 leave the last rows of a tile idle.  Tensor maps over [width, heads, tokens] read the rows where
// they lie, whatever the strides, and give zeros behind a width that is no multiple of 64.
//
// Sequences.  A block finds its own tile: with f(p) = the number of tiles at place p or later of their sequences (counted in tiles from the first
// key that a sequence's queries see), block u works on the place p with f(p + 1) <= u < f(p).  So the tiles with the longest loops of ALL
// sequences start first, and neither the host nor another kernel lays out a plan.  The grid is the bound that the host knows (rows / tile + sequences); the blocks left over fill the rows behind the
// last sequence with zeros.  Rows of a tile behind its sequence's end belong to somebody else: as rows of the result they are not
// stored, as summed rows (V; K of dq; Q and dO of the key gradients) they are set to zero in shared memory, since a weight of zero does not
// silence a NaN.
//
// Forward: one block per pair of query tiles.  A warp loads, a thread per query tile issues its products, a warpgroup per query tile (thread <->
// row <-> TMEM lane) does the softmax: P goes back to TMEM as an operand, O stays there and is rescaled only when a row's maximum has grown by
// 2^8 (2^24 would save 2 to 10 % of the forward and take the errors below from 2.45e-3 to 2.52e-3).
// Backward: two kernels with seven products, after a small one for delta, instead of one with five.  One kernel has a fixed set of columns too
// few (S, dP, dK, dV and dQ of 128 columns are 640 of 512) and adds dQ across blocks with atomics, in an order that changes from run to run; in
// two, P and dS of either orientation are operands in TMEM that never pass through shared memory, every sum has one owner, and the bits are the
// same each time.
//   delta  rows of o and do, read once
//   dq     block per query tile, loops over key tiles:   S = Q K', dP = dO V', dQ += dS K
//   dk dv  block per key tile, loops over query tiles:   S' = K Q', dP' = V dO', dV += P' dO, dK += dS' Q
// The issuing threads take the products in a fixed order (the bits are the same each time) in which each has its operands before the one in front
// of it is done; a product that overwrites columns is issued after the commit of the one that reads them.  One thread that polled for
// whatever was ready first spent more time on polling than the products took (forward 2100 cycles a 128 x 128 tile).
// Query tiles of the key gradients run from the last one down: blocks of one sequence then read the same rows at the same time, out of L2.
//
// Measured in bf16 on documents of 16384 tokens in all (6000 the longest), 32 heads over 8, 128 wide: forward 650 to 840 us, delta 71 to 77, dq 800 to
// 950, dk and dv 1000 to 1140, as the clock goes under the power limit (1.3 ms of products at the library's rate).  What bounds them, widths 128:
//   forward  1450 cycles for 64 keys of both query tiles: a softmax warp's chain (two warps a scheduler; exponentials 1024, products 1284)
//   dq       1800 cycles a 128 x 128 tile, 1536 of products;  dk dv  2960, 2560 of products (two of the four read both operands from shared memory)
// and 12000 cycles a block before the first and after the last tile, which the next block on the SM does not cover.
//
// Roundings to 16 bits: P and dS, as operands of their products.  o is divided by a sum in which the largest weight of every 64 keys counts as it
// was rounded, so that what rounding adds to it moves o only by that key's distance from it: no weight is 1 while the maximum that it is taken
// against lags, and a row that settles on one key was off by up to 2^-9 of itself.  (The sum of all weights as rounded gives the same errors to
// within 1 % and takes 20 % more of the forward's time.)  delta takes o before its rounding (the forward keeps what that takes away, in 16 bits
// more).  Both because an error of o is added to every ds of a row with one sign: dq and dk of rows that settle on few keys are off by 2.45e-3 of
// their norms, where the roundings of dS and of the result itself make 2.4e-3; 3.0e-3 with the sum of unrounded weights, 4.0e-3 with the
// rounded o too.  Maxima, sums, scores, deltas and all accumulators are fp32.
//
// fp16's range is too short for p and dS of any size: both are scaled by powers of two to all of it.  p <= 1 counts 2^14 times.  do v' and delta,
// an average of them, are at most |do| max |v| (Euclidean norms, the keys of the row's sequence and key head), so dS is below 2^14 with the power
// that brings twice that bound under one: |do| is the row's own for dq, and for dk, whose sum goes over rows, the largest of the sequence and key
// head.  A factor of nearly four is left below 65504 for what roundings add, and what falls below the range is less than 2^-37 of |do| max |v|.  No
// sequence and no key head depends on another's gradients.
#include <cuda_fp16.h>

#include "few_rows.cuh"
#include "fp32_pair.cuh"

namespace cm {
namespace packed {
namespace {

constexpr int TILE = 128;
constexpr int PART = 64;                     // columns of scores that are multiplied and waited for as one
constexpr int SLAB = 128 * 128;              // bytes of one [128 rows x 64 columns] slab, 128-byte swizzle
constexpr float RESCALE_AT = 8.f;            // log2
constexpr float FP16_UP = 7.f;               // log2: fp16 weights lie this far above their reference's, for more of the range below them (2^15 at most)

// ---- products --------------------------------------------------------------------------------------------------------
__host__ __device__ constexpr uint32_t idesc(bool half, int n, bool b_mn) {        // M 128, A K-major
  return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(TILE >> 4) << 24);
}
// Descriptors of a slab, to whose low word the steps below are added: one base for an operand, since both orientations have the same row pitch
__device__ __forceinline__ uint64_t base_k(uint32_t tile) { return umma_desc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t base_mn(uint32_t tile) { return umma_desc_sw128(tile, SLAB, 1024); }
// 16-column step k of a K-major operand whose slabs lie one after the other; 16-row step k of the same slabs read MN-major
__device__ __forceinline__ constexpr uint32_t step_k(int k) { return uint32_t((k >> 2) * SLAB + (k & 3) * 32) >> 4; }
__device__ __forceinline__ constexpr uint32_t step_mn(int k) { return uint32_t(k * 2048) >> 4; }
// A in TMEM (row = lane, two 16-bit values of K per column)
__device__ __forceinline__ void umma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// eight floats in a row of shared memory times four, on their way before the next wait
__device__ __forceinline__ void lds_row(float4 (&v)[8], const float* src) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[i].x), "=f"(v[i].y), "=f"(v[i].z), "=f"(v[i].w) : "r"(smem_u32(src + 4 * i)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
  return d;
}
template <bool HALF>
__device__ __forceinline__ uint32_t pair(float lo, float hi) {
  if (!HALF) return pack_bf16(lo, hi);
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool HALF>
__device__ __forceinline__ float2 unpair(uint32_t v) {
  if (!HALF) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
__device__ __forceinline__ void tma_rows(void* dst, const CUtensorMap* map, uint64_t* bar, int col, int head, int row) {
  tma_load_3d(dst, map, bar, col, head, row);
}

// ---- waits -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
}
// A place in a ring of slots, and the parity of its round
template <int SLOTS>
struct Ring {
  int at = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++at == SLOTS) { at = 0; round ^= 1; }
  }
};

// setup_barrier, where warp 0 looks for the block's tile: another warp reads the error word meanwhile
__device__ __forceinline__ bool set_up(const int* err) {
  return __syncthreads_or(threadIdx.x == 64 && err && *reinterpret_cast<const volatile int*>(err) != 0);
}

// ---- sequences -------------------------------------------------------------------------------------------------------
struct Args {
  const int *cu_q, *cu_k;
  int n, T, Tk;                              // sequences, rows of queries and of keys
  int heads, kv_heads;
  int hb, chunks, tok;                       // heads of a tile, tiles of heads in a group, tokens of a tile
  int by_hb;                                 // r / hb is r * by_hb >> 16 for r < 128
  int dim, vdim;
  int units;                                 // blocks per (key head, chunk)
  int splits;                                // forward: blocks that share the keys of a pair of query tiles
  float* part;                               // what each of them leaves: [unit, key head, chunk][split][tile][DV + 3][128 rows]
  float scale, scale_log2;
  void* out;                                 // forward: o [T, heads, vdim]; backward: dq [T, heads, dim] or dk [Tk, kv_heads, dim]
  void* out2;                                // forward: what rounding took from o, or null; backward: dv [Tk, kv_heads, vdim]
  const void *o, *o_rest, *go;               // backward, for delta: o, what rounding took from it (both packed), do with its strides
  long long go_tok, go_head;
  float* lse;                                // [T, heads]: log2 of the sum of weights; +inf without keys; null: not wanted
  float* delta;                              // [T, heads]
  const void* v;                             // backward in fp16, for the bounds of dS: the values with their strides
  long long v_tok, v_head;
  float* big;                                // [T, heads]: |do| of a row
  uint32_t *top, *vtop;                      // [sequences, kv_heads]: the largest finite |do| and |v|, as bits
  int* err;
};

struct Unit {
  int seq, place, total;                     // sequence; place of the tile in it; tiles of all sequences
  int q0, L, k0, Lk;                         // the sequence's queries and keys
  int bad;
};

// Which tile is block u's?  One warp; `per` rows a tile of the sequences' queries or (of_keys) keys.
__device__ Unit find_unit(const Args& a, bool of_keys, int per, int u, int lane) {
  constexpr int KEPT = 4;                    // sequences that a lane keeps the tiles of; more are counted again each time
  Unit r = {};
  bool bad = false;
  int kept[KEPT], ahead[KEPT], q0 = 0, L = 0, k0 = 0, Lk = 0;              // of sequence `lane`
  auto tiles = [&](int rows) { return int(unsigned(rows + per - 1) / unsigned(per)); };
  const int* cu = of_keys ? a.cu_k : a.cu_q;
  auto tiles_of = [&](int i) { return tiles(__ldg(cu + i + 1) - __ldg(cu + i)); };
  // a sequence's first place: the keys before its first query, in tiles
  auto first_of = [&](int rows, int keys) { return of_keys || keys <= rows ? 0 : int(unsigned(keys - rows) / unsigned(per)); };
  auto first_at = [&](int i) { return first_of(__ldg(a.cu_q + i + 1) - __ldg(a.cu_q + i), __ldg(a.cu_k + i + 1) - __ldg(a.cu_k + i)); };
#pragma unroll
  for (int c = 0; c < KEPT; ++c) {
    const int i = c * 32 + lane;
    kept[c] = ahead[c] = 0;
    if (c * 32 >= a.n) continue;
    if (i < a.n) {
      const int x0 = __ldg(a.cu_q + i), x1 = __ldg(a.cu_q + i + 1), y0 = __ldg(a.cu_k + i), y1 = __ldg(a.cu_k + i + 1);
      bad |= x0 < 0 || x1 < x0 || x1 > a.T || y0 < 0 || y1 < y0 || y1 > a.Tk || (i == 0 && (x0 != 0 || y0 != 0));
      kept[c] = tiles(of_keys ? y1 - y0 : x1 - x0);
      ahead[c] = first_of(x1 - x0, y1 - y0);
      if (c == 0) { q0 = x0; L = x1 - x0; k0 = y0; Lk = y1 - y0; }
    }
  }
  if (a.n == 0) bad = __ldg(a.cu_q) != 0 || __ldg(a.cu_k) != 0;
  for (int i = KEPT * 32 + lane; i < a.n; i += 32) {
    const int x0 = __ldg(a.cu_q + i), x1 = __ldg(a.cu_q + i + 1), y0 = __ldg(a.cu_k + i), y1 = __ldg(a.cu_k + i + 1);
    bad |= x0 < 0 || x1 < x0 || x1 > a.T || y0 < 0 || y1 < y0 || y1 > a.Tk;
  }
  r.bad = __any_sync(0xffffffffu, bad);
  if (r.bad) return r;
  auto after = [&](int p) {                  // tiles at place p or later
    int s = 0;
#pragma unroll
    for (int c = 0; c < KEPT; ++c) s += min(kept[c], max(0, ahead[c] + kept[c] - p));
    for (int i = KEPT * 32 + lane; i < a.n; i += 32) s += min(tiles_of(i), max(0, first_at(i) + tiles_of(i) - p));
    return __reduce_add_sync(0xffffffffu, s);
  };
  int most = max(max(ahead[0] + kept[0], ahead[1] + kept[1]), max(ahead[2] + kept[2], ahead[3] + kept[3]));
  for (int i = KEPT * 32 + lane; i < a.n; i += 32) most = max(most, first_at(i) + tiles_of(i));
  r.total = after(0);
  if (u >= r.total) return r;
  int lo = 0, hi = __reduce_max_sync(0xffffffffu, most), from_hi = 0;         // after(lo) > u >= after(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, f = after(mid);
    if (f > u) lo = mid;
    else { hi = mid; from_hi = f; }
  }
  int rank = u - from_hi, seq = 0;           // hi is lo + 1: the rank-th of the sequences that have a tile at this place
  for (int c = 0, i0 = 0; i0 < a.n; i0 += 32, ++c) {
    const bool there = i0 + lane < a.n;
    const int t = c == 0 ? kept[0] : c == 1 ? kept[1] : c == 2 ? kept[2] : c == 3 ? kept[3] : there ? tiles_of(i0 + lane) : 0;
    const int f = c == 0 ? ahead[0] : c == 1 ? ahead[1] : c == 2 ? ahead[2] : c == 3 ? ahead[3] : there ? first_at(i0 + lane) : 0;
    const bool at = f <= lo && lo < f + t;
    const unsigned has = __ballot_sync(0xffffffffu, at);
    if (rank < __popc(has)) {
      const int src = __ffs(__ballot_sync(0xffffffffu, at && __popc(has & ((1u << lane) - 1)) == rank)) - 1;
      seq = i0 + src;
      r.place = lo - __shfl_sync(0xffffffffu, f, src);
      break;
    }
    rank -= __popc(has);
  }
  r.seq = seq;
  if (seq < 32) {
    r.q0 = __shfl_sync(0xffffffffu, q0, seq); r.L = __shfl_sync(0xffffffffu, L, seq);
    r.k0 = __shfl_sync(0xffffffffu, k0, seq); r.Lk = __shfl_sync(0xffffffffu, Lk, seq);
  } else {
    r.q0 = __ldg(a.cu_q + seq); r.L = __ldg(a.cu_q + seq + 1) - r.q0;
    r.k0 = __ldg(a.cu_k + seq); r.Lk = __ldg(a.cu_k + seq + 1) - r.k0;
  }
  return r;
}

// The blocks left over: zeros into the rows [begin, rows) of a [rows, heads, width] result, columns of `heads` heads from head0 on
__device__ void clear_rows(void* out, int begin, int rows, int all_heads, int head0, int heads, int width, int part, int parts) {
  const int pieces = heads * width / 8;
  for (long long r = begin + part; r < rows; r += parts) {
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + (r * all_heads + head0) * width);
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) dst[i] = make_uint4(0, 0, 0, 0);
  }
}

// rows [from, 128) of `slabs` slabs set to zero by one warp
__device__ __forceinline__ void clear_tail(uint8_t* tile, int slabs, int from, int lane) {
  for (int s = 0; s < slabs; ++s)
    for (int i = from * 8 + lane; i < TILE * 8; i += 32) reinterpret_cast<uint4*>(tile + s * SLAB)[i] = make_uint4(0, 0, 0, 0);
}

// copies in flight land before the shared memory is released
__device__ __forceinline__ void settle(volatile int* abort_flag) {
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
    __syncthreads();
  }
}

// 32 fp32 columns as 16-bit values, to columns col .. col + 31 of row r of slabs in shared memory
template <bool HALF>
__device__ __forceinline__ void put_columns(uint8_t* slabs, int r, int col, const uint32_t (&x)[32]) {
  uint8_t* row = slabs + (col >> 6) * SLAB + r * 128;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 o;
    o.x = pair<HALF>(__uint_as_float(x[q * 8]), __uint_as_float(x[q * 8 + 1]));
    o.y = pair<HALF>(__uint_as_float(x[q * 8 + 2]), __uint_as_float(x[q * 8 + 3]));
    o.z = pair<HALF>(__uint_as_float(x[q * 8 + 4]), __uint_as_float(x[q * 8 + 5]));
    o.w = pair<HALF>(__uint_as_float(x[q * 8 + 6]), __uint_as_float(x[q * 8 + 7]));
    *reinterpret_cast<uint4*>(row + ((((col >> 3) + q) & 7) ^ (r & 7)) * 16) = o;
  }
}
// Which rows of a tile a lane sends with LANES lanes a row: their places behind the tile's first row of the result in steps of the result's width,
// -1 for those that are not stored
template <int LANES, typename PlaceOf>
__device__ __forceinline__ void places(int (&at)[LANES], int row0, int lane, PlaceOf place_of) {
#pragma unroll
  for (int i = 0; i < LANES; ++i) at[i] = place_of(row0 + i * (32 / LANES) + lane / LANES);
}
// The warp's 32 rows of one slab (64 columns), its columns as columns begin .. begin + 8 LANES - 1 of the result, of whose `width` that exist: whole
// lines, where each thread for itself would store 16 bytes of 32 rows at a time
template <int LANES>
__device__ __forceinline__ void send_rows(const uint8_t* slab, int row0, int begin, int width, int lane, const int (&at)[LANES], uint16_t* out) {
  __syncwarp();
  const int piece = begin / 8 + lane % LANES;
  const bool exists = piece * 8 < width;
  uint4 v[LANES];
#pragma unroll
  for (int i = 0; i < LANES; ++i) {
    const int r = row0 + i * (32 / LANES) + lane / LANES;
    v[i] = *reinterpret_cast<const uint4*>(slab + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
  }
  out += piece * 8;
#pragma unroll
  for (int i = 0; i < LANES; ++i)
    if (at[i] >= 0 && exists) *reinterpret_cast<uint4*>(out + (long long)at[i] * width) = v[i];
  __syncwarp();
}

// 32 fp32 columns less what put_columns makes of them
template <bool HALF>
__device__ __forceinline__ void take_rest(uint32_t (&x)[32]) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 v = make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
    const uint32_t w = pair<HALF>(v.x, v.y);
    const float2 u = HALF ? unpair<HALF>(w) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    x[e] = __float_as_uint(v.x - u.x);
    x[e + 1] = __float_as_uint(v.y - u.y);
  }
}

struct Masked { static constexpr bool value = true; };
struct Whole { static constexpr bool value = false; };

// ---- forward ---------------------------------------------------------------------------------------------------------
// Eight compute warps, two that issue products, one that loads.  One issuing thread for all products of a block was the longest chain of the backward:
// a wait that has nothing to wait for and eight products cost it 250 cycles beside the compute warps (dq 2110 cycles a 128 x 128 tile, 1800 with two).
constexpr int THREADS = 352;
constexpr int MMA_WARP = 8, TMA_WARP = 10;

// Few rows on many keys: the key tiles of a pair of query tiles are shared out among neighbouring blocks, no fewer than four to each, and
// join_kernel makes one result of what they leave.
struct Share {
  int begin, tiles, pieces;                  // first key tile, key tiles of a block, blocks that have any
};
constexpr int FEWEST_TILES = 4;              // 512 keys: about as long as a block's set-up and what it leaves take
__device__ __forceinline__ Share share_of(const Args& a, const Unit& unit, int split) {
  const int last = min(unit.L, 2 * (unit.place + 1) * a.tok) - 1 + unit.Lk - unit.L;       // last key that the pair sees
  const int all = last >= 0 ? last / TILE + 1 : 0;
  Share s;
  s.tiles = a.splits == 1 ? max(all, 1) : max(FEWEST_TILES, (all + a.splits - 1) / a.splits);
  s.pieces = max(1, (all + s.tiles - 1) / s.tiles);
  s.begin = split * s.tiles;
  return s;
}

template <int D, int DV>
struct Fwd {
  static constexpr int KS = D / 64, VS = DV / 64;
  static constexpr int K_SLOTS = 3, V_SLOTS = DV == 128 ? 2 : 3;
  struct Shared {
    uint64_t q_full[2], k_full[K_SLOTS], k_empty[K_SLOTS], v_full[V_SLOTS], v_empty[V_SLOTS], tail;
    uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];       // query tile, half of the key tile
    Unit unit;
    uint32_t tmem_slot;
    int abort_flag;
  };
  static constexpr int SMEM = (2 * KS + K_SLOTS * KS + V_SLOTS * VS) * SLAB + (int)sizeof(Shared) + 1024;
};

template <bool HALF, int D, int DV>
__global__ void __launch_bounds__(THREADS, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const Args a) {
  using F = Fwd<D, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * F::KS * SLAB;
  uint8_t* sV = sK + F::K_SLOTS * F::KS * SLAB;
  auto* sh = reinterpret_cast<typename F::Shared*>(sV + F::V_SLOTS * F::VS * SLAB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  few::let_next_start();
  const int tiles = blockIdx.x / a.splits, split = blockIdx.x % a.splits;             // two query tiles; a share of their keys
  const int hh = a.kv_heads * a.chunks, u = tiles / hh, kvh = (tiles % hh) / a.chunks, chunk = tiles % a.chunks;
  const int head0 = kvh * (a.heads / a.kv_heads) + chunk * a.hb;
  volatile int* abort_flag = &sh->abort_flag;
  if (warp == 0) {
    const Unit r = find_unit(a, false, 2 * a.tok, u, lane);
    if (lane == 0) sh->unit = r;
  }
  if (tid == 32) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->q_full[t], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh->s_full[t][b], 1);
        mbar_init(&sh->p_full[t][b], 4);
        mbar_init(&sh->pv_done[t][b], 1);
      }
    }
    for (int s = 0; s < F::K_SLOTS; ++s) { mbar_init(&sh->k_full[s], 1); mbar_init(&sh->k_empty[s], 2); }
    for (int s = 0; s < F::V_SLOTS; ++s) { mbar_init(&sh->v_full[s], 1); mbar_init(&sh->v_empty[s], 2); }
    mbar_init(&sh->tail, 1);
    sh->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) { tmem_alloc(&sh->tmem_slot, 512); tmem_relinquish(); }
  if (warp == TMA_WARP && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  const bool drain = set_up(a.err);
  tc_fence_after();
  const uint32_t tmem = sh->tmem_slot;       // S_t at 128 t, one half of it after the other, P over the half it came from; O_t at 256 + DV t
  const Unit unit = sh->unit;
  if (drain || unit.bad || u >= unit.total) {
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
    if (drain) return;
    if (unit.bad) {
      if (tid == 0 && a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
      return;
    }
    if (split == 0) clear_rows(a.out, __ldg(a.cu_q + a.n), a.T, a.heads, head0, a.hb, a.vdim, u - unit.total, a.units - unit.total);
    return;
  }
  // this block's key tiles; from here on the keys are counted from the first of them
  const Share share = share_of(a, unit, split);
  const int q0 = unit.q0, L = unit.L, k0 = unit.k0 + share.begin * TILE, Lk = unit.Lk - share.begin * TILE;
  const int off = Lk - L;                    // query i sees the keys up to i + off
  const int rows = a.hb * a.tok;
  if (split > 0 && split >= share.pieces) {
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
    return;
  }
  // halves of key tiles (64 keys) of query tile t, and the first of them that the mask cuts
  int n[2], whole[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = (2 * unit.place + t) * a.tok, last = min(L, first + a.tok) - 1;
    n[t] = first < L && off + last >= 0 ? min((off + last) / PART + 1, 2 * share.tiles) : 0;
    whole[t] = off + first + 1 > 0 ? (off + first + 1) / PART : 0;
  }
  const int most = (max(n[0], n[1]) + 1) / 2;

  if (warp == TMA_WARP) {
    // ------------------------------ loads ------------------------------
    bool ok = true;
    auto load_q = [&](int t) {
      if (n[t] == 0 || lane != 0) return;
      mbar_expect_tx(&sh->q_full[t], F::KS * rows * 128);
      for (int s = 0; s < F::KS; ++s)
        tma_rows(sQ + (t * F::KS + s) * SLAB, &tmQ, &sh->q_full[t], s * 64, head0, q0 + (2 * unit.place + t) * a.tok);
    };
    load_q(0);
    for (int j = 0; j < most && ok; ++j) {
      const int ks = j % F::K_SLOTS, vs = j % F::V_SLOTS;
      ok = warp_wait(&sh->k_empty[ks], ((j / F::K_SLOTS) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&sh->k_full[ks], F::KS * SLAB);
        for (int s = 0; s < F::KS; ++s) tma_rows(sK + (ks * F::KS + s) * SLAB, &tmK, &sh->k_full[ks], s * 64, kvh, k0 + j * TILE);
      }
      if (j == 0) load_q(1);
      ok = warp_wait(&sh->v_empty[vs], ((j / F::V_SLOTS) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      const bool cut = (j + 1) * TILE > Lk;                   // the sequence's last tile: the rows behind its end are set to zero
      uint64_t* bar = cut ? &sh->tail : &sh->v_full[vs];
      if (lane == 0) {
        mbar_expect_tx(bar, F::VS * SLAB);
        for (int s = 0; s < F::VS; ++s) tma_rows(sV + (vs * F::VS + s) * SLAB, &tmV, bar, s * 64, kvh, k0 + j * TILE);
      }
      if (cut) {
        ok = warp_wait(bar, 0, abort_flag, a.err, ERR_WAIT_FULL);
        if (!ok) break;
        clear_tail(sV + vs * F::VS * SLAB, F::VS, Lk - j * TILE, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->v_full[vs]);
      }
    }
  } else if (warp >= MMA_WARP) {
    // ------------------------------ products of query tile t ------------------------------
    if (elect_one()) {
      constexpr uint32_t id_s = idesc(HALF, PART, false), id_o = idesc(HALF, DV, true);
      const int t = warp - MMA_WARP, count = t ? n[1] : n[0];
      const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * DV;
      const uint64_t dQ = base_k(smem_u32(sQ + t * F::KS * SLAB)), dK = base_k(smem_u32(sK)), dV = base_mn(smem_u32(sV));
      Ring<F::K_SLOTS> rk;
      Ring<F::V_SLOTS> rv;
      bool ok = true;
      auto scores = [&](int j) {             // S(j) = Q K(j)', 64 keys; a key tile is let go after its second half
        if (!(j & 1)) ok = mbar_wait(&sh->k_full[rk.at], rk.round, abort_flag, a.err, ERR_WAIT_FULL);
        if (!ok) return;
        tc_fence_after();
        const uint64_t d = dK + rk.at * (F::KS * SLAB >> 4) + (j & 1) * (SLAB / 2 >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) umma_f16(tS + (j & 1) * 64, dQ + step_k(k), d + step_k(k), id_s, k != 0);
        umma_commit(&sh->s_full[t][j & 1]);
        if ((j & 1) || j + 1 == count) {
          umma_commit(&sh->k_empty[rk.at]);
          rk.next();
        }
      };
      if (count > 0) ok = mbar_wait(&sh->q_full[t], 0, abort_flag, a.err, ERR_WAIT_FULL);
      if (ok && count > 0) scores(0);
      if (ok && count > 1) scores(1);
      for (int j = 0; j < count && ok; ++j) {
        if (!(j & 1)) ok = mbar_wait(&sh->v_full[rv.at], rv.round, abort_flag, a.err, ERR_WAIT_FULL);
        ok = ok && mbar_wait(&sh->p_full[t][j & 1], (j >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint64_t d = dV + rv.at * (F::VS * SLAB >> 4) + (j & 1) * step_mn(4);
#pragma unroll
        for (int k = 0; k < PART / 16; ++k) umma_ta(tO, tS + (j & 1) * 64 + k * 8, d + step_mn(k), id_o, (j | k) != 0);
        umma_commit(&sh->pv_done[t][j & 1]);
        if ((j & 1) || j + 1 == count) {
          umma_commit(&sh->v_empty[rv.at]);
          rv.next();
        }
        if (j + 2 < count) {                 // over the columns of P(j)
          ok = mbar_wait(&sh->pv_done[t][j & 1], (j >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
          if (ok) scores(j + 2);
        }
      }
      // key tiles that the other query tile alone looks at
      for (int j = (count + 1) / 2; j < most && ok; ++j) {
        ok = mbar_wait(&sh->k_full[rk.at], rk.round, abort_flag, a.err, ERR_WAIT_FULL) &&
             mbar_wait(&sh->v_full[rv.at], rv.round, abort_flag, a.err, ERR_WAIT_FULL);
        if (!ok) break;
        mbar_arrive(&sh->k_empty[rk.at]);
        mbar_arrive(&sh->v_empty[rv.at]);
        rk.next();
        rv.next();
      }
    }
  } else {
    // ------------------------------ softmax of query tile t ------------------------------
    const int t = warp >> 2, r = tid & 127, tok = r * a.by_hb >> 16, qt = 2 * unit.place + t;
    const int pos = qt * a.tok + tok;                         // position of this row's query
    const bool mine = r < rows && pos < L;
    const int last = mine ? off + pos : -1;                   // last key it sees
    const uint32_t lane_addr = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + 256 + t * DV + lane_addr;
    float m_ref = -INFINITY, l = 0.f, gained = 0.f;           // sums of the weights, and of what rounding adds to the largest ones
    auto part = [&](int j, auto where) {
      constexpr bool MASK = decltype(where)::value;
      const int lim = last - j * PART;                        // columns up to lim are seen
      const uint32_t tS = tmem + t * 128 + (j & 1) * 64 + lane_addr;
      if (!warp_wait(&sh->s_full[t][j & 1], (j >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
      uint32_t s0[32], s1[32];
      tmem_ld_32x32(tS, s0);
      tmem_ld_32x32(tS + 32, s1);
      tmem_ld_wait();
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const int to = e >> 1 & 1;
        top[to] = max3(top[to], !MASK || e <= lim ? __uint_as_float(s0[e]) : -INFINITY, !MASK || e + 1 <= lim ? __uint_as_float(s0[e + 1]) : -INFINITY);
        top[2 + to] = max3(top[2 + to], !MASK || 32 + e <= lim ? __uint_as_float(s1[e]) : -INFINITY,
                           !MASK || 33 + e <= lim ? __uint_as_float(s1[e + 1]) : -INFINITY);
      }
      const float largest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const float m_new = largest != -INFINITY ? largest * a.scale_log2 : -INFINITY;            // a scale of zero leaves "nothing seen" as it is
      float alpha = 1.f;
      constexpr float UP = HALF ? FP16_UP : 0.f;
      if (m_new > m_ref + (RESCALE_AT + UP)) {                // also from -inf
        alpha = ex2(m_ref - (m_new - UP));
        m_ref = m_new - UP;
        l *= alpha;
        gained *= alpha;
      }
      if (__any_sync(0xffffffffu, alpha != 1.f) && j > 0) {   // O of all parts before this one
        if (!warp_wait(&sh->pv_done[t][(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < DV / 32; c += 2) {
          uint32_t o[2][32];
          tmem_ld_32x32(tO + c * 32, o[0]);
          tmem_ld_32x32(tO + c * 32 + 32, o[1]);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[h][e] = __float_as_uint(__uint_as_float(o[h][e]) * alpha);
            tmem_st(tO + (c + h) * 32, o[h]);
          }
        }
      }
      const float ref = m_ref == -INFINITY ? 0.f : m_ref;     // nothing seen so far
      Pair sum[2] = {pr(0.f), pr(0.f)};
      uint32_t p[32];
      auto quarter = [&](const uint32_t (&sc)[32], int col0, int at) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 z = pr_get(pr_fma(pr(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), pr(a.scale_log2), pr(-ref)));
          float x = ex2(z.x), y = ex2(z.y);
          if (MASK) {
            x = col0 + 2 * e <= lim ? x : 0.f;
            y = col0 + 2 * e + 1 <= lim ? y : 0.f;
          }
          sum[e & 1] = sum[e & 1] + pr(x, y);
          p[at + e] = pair<HALF>(x, y);
        }
      };
      quarter(s0, 0, 0);
      quarter(s1, 32, 16);
      tmem_st(tS, p);
      l += pr_sum(sum[0] + sum[1]);
      if (largest != -INFINITY) {                             // the part's largest weight, as above
        const float x = ex2(fmaf(largest, a.scale_log2, -ref));
        gained += unpair<HALF>(pair<HALF>(x, 0.f)).x - x;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->p_full[t][j & 1]);
      return true;
    };
    const int count = t ? n[1] : n[0], open = t ? whole[1] : whole[0];
    bool ok = true;
    for (int j = 0; j < min(count, open) && ok; ++j) ok = part(j, Whole{});
    for (int j = min(count, open); j < count && ok; ++j) ok = part(j, Masked{});
    if (ok && count > 0) ok = warp_wait(&sh->pv_done[t][(count - 1) & 1], ((count - 1) >> 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL);
    if (ok) {
      tc_fence_after();
      if (share.pieces > 1) {
        float* to = a.part + (((long long)blockIdx.x * 2 + t) * (DV + 3)) * TILE + r;
        to[0] = m_ref;
        to[TILE] = l;
        to[2 * TILE] = l + gained;
#pragma unroll
        for (int c = 0; c < DV / 32; ++c) {
          uint32_t o[32];
          if (count > 0) {
            tmem_ld_32x32(tO + c * 32, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) to[(3 + c * 32 + e) * TILE] = last >= 0 ? __uint_as_float(o[e]) : 0.f;            // nothing seen here
        }
      } else {
        const float taken = l + gained, inv = taken > 0.f ? 1.f / taken : taken == 0.f ? 0.f : taken;            // a NaN stays
        const long long at = (long long)(q0 + pos) * a.heads + head0 + (r - tok * a.hb);
        const float f = last >= 0 ? inv : 0.f;
        uint8_t* stage = sQ + t * F::KS * SLAB;                 // Q_t has been used
        int places_at[8];
        places(places_at, (warp & 3) * 32, lane, [&](int r) {
          const int tok = r * a.by_hb >> 16;
          return r < rows && qt * a.tok + tok < L ? tok * a.heads + (r - tok * a.hb) : -1;
        });
        const long long first = ((long long)(q0 + qt * a.tok) * a.heads + head0) * a.vdim;
        // o to one slab and what its rounding takes away to the other, 64 columns at a time; where Q_t has one slab alone (width 64) one after the other
        constexpr int PASSES = F::KS == 1 ? 2 : 1;
  #pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
          if (pass == 1 && !a.out2) break;
  #pragma unroll
          for (int c = 0; c < DV / 32; ++c) {
            uint32_t o[32];
            if (count > 0) {
              tmem_ld_32x32(tO + c * 32, o);
              tmem_ld_wait();
            }
  #pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = last >= 0 ? __float_as_uint(__uint_as_float(o[e]) * f) : 0u;            // a row without keys
            if (pass == 0) put_columns<HALF>(stage, r, (c & 1) * 32, o);
            if (a.out2 && pass == PASSES - 1) {
              take_rest<HALF>(o);
              put_columns<HALF>(stage + (PASSES == 1 ? SLAB : 0), r, (c & 1) * 32, o);
            }
            if (c & 1) {
              const int begin = (c - 1) * 32;
              if (pass == 0) send_rows(stage, (warp & 3) * 32, begin, a.vdim, lane, places_at, reinterpret_cast<uint16_t*>(a.out) + first);
              if (a.out2 && pass == PASSES - 1)
                send_rows(stage + (PASSES == 1 ? SLAB : 0), (warp & 3) * 32, begin, a.vdim, lane, places_at, reinterpret_cast<uint16_t*>(a.out2) + first);
            }
          }
        }
        if (mine && a.lse) a.lse[at] = l == 0.f ? INFINITY : m_ref + log2f(l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  settle(abort_flag);
  if (warp == MMA_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// What the blocks of a pair of query tiles left, in the order of their keys.  A block per tile and eight columns, a thread per row.
template <bool HALF, int DV>
__global__ void __launch_bounds__(TILE) packed_join_kernel(const Args a) {
  constexpr int COLUMNS = 8, STEP = (DV + 3) * TILE * 2;
  __shared__ Unit found;
  const int chunks_of = DV / COLUMNS, c0 = blockIdx.x % chunks_of * COLUMNS, t = blockIdx.x / chunks_of % 2, tiles = blockIdx.x / chunks_of / 2;
  const int hh = a.kv_heads * a.chunks, u = tiles / hh, kvh = (tiles % hh) / a.chunks, chunk = tiles % a.chunks, r = threadIdx.x;
  if (threadIdx.x < 32) {
    const Unit f = find_unit(a, false, 2 * a.tok, u, threadIdx.x);
    if (threadIdx.x == 0) found = f;
  }
  __syncthreads();
  const Unit unit = found;
  few::wait_for_input();                     // by every block: the next kernel of the stream counts on this one having waited
  if (unit.bad || u >= unit.total || c0 >= a.vdim) return;
  const int pieces = share_of(a, unit, 0).pieces, tok = r * a.by_hb >> 16, pos = (2 * unit.place + t) * a.tok + tok;
  if (pieces == 1 || r >= a.hb * a.tok || pos >= unit.L) return;
  const float* from = a.part + ((long long)tiles * a.splits * 2 + t) * (DV + 3) * TILE + r;
  float m = -INFINITY, l = 0.f, taken = 0.f, o[COLUMNS] = {};
  for (int s = 0; s < pieces; ++s) m = fmaxf(m, from[(long long)s * STEP]);
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 2
  for (int s = 0; s < pieces; ++s) {
    const float* x = from + (long long)s * STEP;
    const float by = ex2(x[0] - ref);
    l += by * x[TILE];
    taken += by * x[2 * TILE];
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) o[c] += by * x[(3 + c0 + c) * TILE];
  }
  const float inv = taken > 0.f ? 1.f / taken : taken == 0.f ? 0.f : taken;               // a NaN stays
  const long long at = (long long)(unit.q0 + pos) * a.heads + kvh * (a.heads / a.kv_heads) + chunk * a.hb + (r - tok * a.hb);
  uint32_t w[4], rest[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float x = o[2 * c] * inv, y = o[2 * c + 1] * inv;
    w[c] = pair<HALF>(x, y);
    const float2 f = unpair<HALF>(w[c]);
    rest[c] = pair<HALF>(x - f.x, y - f.y);
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + at * a.vdim + c0) = make_uint4(w[0], w[1], w[2], w[3]);
  if (a.out2) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out2) + at * a.vdim + c0) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
  if (a.lse && c0 == 0) a.lse[at] = l == 0.f ? INFINITY : m + log2f(l);
}

// ---- backward: delta -----------------------------------------------------------------------------------------------------
// delta[i] = do[i] . o[i] before its rounding, in fp16 also |do| of the row.  DV / 8 lanes a row, four rows of a lane on their way at once: three reads
// of a row's width at the memory's rate.  Inside the dq kernel, whose blocks have an SM to themselves, nothing would run meanwhile (9000 cycles a
// block, 120 us at 16384 x 32 rows of 128; here 71).
constexpr int DELTA_THREADS = 256, DELTA_AHEAD = 4;

// the last sequence that begins at or before row `tok`, of n > 0
__device__ __forceinline__ int sequence_of(const int* cu, int n, int tok) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= tok) lo = mid;
    else hi = mid;
  }
  return lo;
}
// 2^14 p is rounded to fp16, and p (do v' - delta) with it
constexpr float P_UP = 14.f, P_DOWN = 1.f / 16384;
// For 2 `bound` in [2^e, 2^(e + 1)): the power 2^-(e + 1), under which it is in [1/2, 1), and its inverse
__device__ __forceinline__ void powers_for(float bound, float& up, float& down) {
  const int e = int(__float_as_uint(2.f * bound) >> 23) - 127;
  const bool usable = bound > 0.f && e > -100 && e < 100;     // |do| and |v| of fp16 rows: 2^-47 to 2^41
  up = usable ? __uint_as_float(uint32_t(126 - e) << 23) : 1.f;
  down = usable ? __uint_as_float(uint32_t(128 + e) << 23) : 1.f;
}

template <bool HALF, int LANES>
__global__ void __launch_bounds__(DELTA_THREADS, 4) packed_delta_kernel(const Args a) {
  constexpr int ROWS = DELTA_THREADS / LANES;
  const int piece = threadIdx.x % LANES;
  // what lies behind the last sequence counts for nothing
  const long long rows = (long long)min(max(__ldg(a.cu_q + a.n), 0), a.T) * a.heads, base = (long long)blockIdx.x * (ROWS * DELTA_AHEAD);
  const long long row0 = base + threadIdx.x / LANES, tok0 = base / a.heads;
  const unsigned head0 = unsigned(base - tok0 * a.heads) + threadIdx.x / LANES;
  uint4 x[DELTA_AHEAD], z[DELTA_AHEAD], y[DELTA_AHEAD];
#pragma unroll
  for (int i = 0; i < DELTA_AHEAD; ++i) {
    const long long row = row0 + i * ROWS;
    x[i] = z[i] = y[i] = make_uint4(0, 0, 0, 0);
    if (row < rows && piece * 8 < a.vdim) {
      const unsigned more = (head0 + i * ROWS) / unsigned(a.heads), head = head0 + i * ROWS - more * a.heads;
      const long long tok = tok0 + more;
      x[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.o) + row * a.vdim) + piece);
      z[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.o_rest) + row * a.vdim) + piece);
      y[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.go) + tok * a.go_tok + head * a.go_head) + piece);
    }
  }
#pragma unroll
  for (int i = 0; i < DELTA_AHEAD; ++i) {
    const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, zs[4] = {z[i].x, z[i].y, z[i].z, z[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
    float dot = 0.f, big = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpair<HALF>(xs[e]), h = unpair<HALF>(zs[e]), g = unpair<HALF>(ys[e]);
      dot = fmaf(f.x + h.x, g.x, fmaf(f.y + h.y, g.y, dot));
      if (HALF) big = fmaf(g.x, g.x, fmaf(g.y, g.y, big));
    }
#pragma unroll
    for (int o = LANES >> 1; o > 0; o >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (HALF) big += __shfl_xor_sync(0xffffffffu, big, o);
    }
    const long long row = row0 + i * ROWS;
    if (piece == 0 && row < rows) {
      a.delta[row] = dot;
      if (HALF) a.big[row] = sqrtf(big);
    }
  }
}

// fp16: the largest |v| and |do| of each sequence and key head.  A warp takes 32 tokens of a key head, most often of one sequence, and reports once for
// each sequence among them (row by row, the few words that all rows ask for took 50 us at 8192 x 32 rows).
template <int LANES>
__global__ void __launch_bounds__(DELTA_THREADS) packed_sizes_kernel(const Args a) {
  constexpr int AT_ONCE = 32 / LANES;
  const int lane = threadIdx.x & 31, piece = lane % LANES, group = a.heads / a.kv_heads;
  const long long warp = (long long)blockIdx.x * (DELTA_THREADS / 32) + (threadIdx.x >> 5), of_v = (long long)((a.Tk + 31) / 32) * a.kv_heads;
  const bool v = warp < of_v;                // the others look at |do|
  const long long mine = v ? warp : warp - of_v;
  const int first = int(mine / a.kv_heads) * 32, kvh = int(mine % a.kv_heads), tok = first + lane;
  const int* cu = v ? a.cu_k : a.cu_q;
  const int rows = min(max(__ldg(cu + a.n), 0), v ? a.Tk : a.T);
  if (first >= rows) return;
  float big = 0.f;
  if (v) {
#pragma unroll
    for (int i = 0; i < LANES; ++i) {
      const int t = first + i * AT_ONCE + lane / LANES;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (t < rows && piece * 8 < a.vdim)
        x = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.v) + t * a.v_tok + kvh * a.v_head) + piece);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpair<true>(xs[e]);
        sum = fmaf(f.x, f.x, fmaf(f.y, f.y, sum));
      }
#pragma unroll
      for (int o = LANES >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float own = __shfl_sync(0xffffffffu, sum, (lane % AT_ONCE) * LANES);
      if (lane / AT_ONCE == i) big = sqrtf(own);
    }
  } else if (tok < rows) {
    for (int h = 0; h < group; ++h) {
      const float x = a.big[(long long)tok * a.heads + kvh * group + h];
      if (isfinite(x)) big = fmaxf(big, x);
    }
  }
  const int seq = tok < rows ? sequence_of(cu, a.n, tok) : -1;
  const uint32_t bits = isfinite(big) ? __float_as_uint(big) : 0u;
  for (unsigned todo = __ballot_sync(0xffffffffu, seq >= 0); todo;) {
    const int s = __shfl_sync(0xffffffffu, seq, __ffs(todo) - 1);
    const uint32_t most = __reduce_max_sync(0xffffffffu, seq == s ? bits : 0u);
    uint32_t* at = (v ? a.vtop : a.top) + (long long)s * a.kv_heads + kvh;
    if (lane == 0 && most > *reinterpret_cast<volatile uint32_t*>(at)) atomicMax(at, most);            // the same in any order
    todo &= ~__ballot_sync(0xffffffffu, seq == s);
  }
}

// ---- backward: query gradients -------------------------------------------------------------------------------------------
template <int D, int DV>
struct Dq {
  static constexpr int KS = D / 64, VS = DV / 64, K_SLOTS = 3, V_SLOTS = 2;
  struct Shared {
    uint64_t q_full, rows_in, k_full[K_SLOTS], k_empty[K_SLOTS], v_full[V_SLOTS], v_empty[V_SLOTS], tail;
    uint64_t s_full[2], s_free[2], dp_full[2], ds_full[2], dq_done[2], acc_done;        // half of the key tile
    Unit unit;
    uint32_t tmem_slot;
    int abort_flag;
  };
  static constexpr int SMEM = (KS + VS + K_SLOTS * KS + V_SLOTS * VS) * SLAB + (int)sizeof(Shared) + 1024;
};

template <bool HALF, int D, int DV>
__global__ void __launch_bounds__(THREADS, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmG, const Args a) {
  using F = Dq<D, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = sQ + F::KS * SLAB;
  uint8_t* sK = sG + F::VS * SLAB;
  uint8_t* sV = sK + F::K_SLOTS * F::KS * SLAB;
  auto* sh = reinterpret_cast<typename F::Shared*>(sV + F::V_SLOTS * F::VS * SLAB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hh = a.kv_heads * a.chunks, u = blockIdx.x / hh, kvh = (blockIdx.x % hh) / a.chunks, chunk = blockIdx.x % a.chunks;
  const int head0 = kvh * (a.heads / a.kv_heads) + chunk * a.hb;
  volatile int* abort_flag = &sh->abort_flag;
  if (warp == 0) {
    const Unit r = find_unit(a, false, a.tok, u, lane);
    if (lane == 0) sh->unit = r;
  }
  if (tid == 32) {
    mbar_init(&sh->q_full, 1);
    for (int s = 0; s < F::K_SLOTS; ++s) { mbar_init(&sh->k_full[s], 1); mbar_init(&sh->k_empty[s], 1); }
    for (int s = 0; s < F::V_SLOTS; ++s) { mbar_init(&sh->v_full[s], 1); mbar_init(&sh->v_empty[s], 1); }
    mbar_init(&sh->rows_in, 8);
    mbar_init(&sh->tail, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->s_full[b], 1);
      mbar_init(&sh->s_free[b], 4);
      mbar_init(&sh->dp_full[b], 1);
      mbar_init(&sh->ds_full[b], 4);
      mbar_init(&sh->dq_done[b], 1);
    }
    mbar_init(&sh->acc_done, 1);
    sh->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) { tmem_alloc(&sh->tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  const bool drain = set_up(a.err);
  tc_fence_after();
  const uint32_t tmem = sh->tmem_slot;       // S at 0, dP at 128 (halves of 64 columns, dS over those of dP), dQ at 256; Q at 384, dO at 448
  const Unit unit = sh->unit;
  if (drain || unit.bad || u >= unit.total) {
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
    if (drain) return;
    if (unit.bad) {
      if (tid == 0 && a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
      return;
    }
    clear_rows(a.out, __ldg(a.cu_q + a.n), a.T, a.heads, head0, a.hb, a.dim, u - unit.total, a.units - unit.total);
    return;
  }
  const int q0 = unit.q0, L = unit.L, k0 = unit.k0, Lk = unit.Lk;
  const int off = Lk - L, rows = a.hb * a.tok, first = unit.place * a.tok, end = min(L, first + a.tok);
  const int n = off + end - 1 >= 0 ? (off + end - 1) / TILE + 1 : 0;
  const int open = off + first + 1 > 0 ? min(n, (off + first + 1) / TILE) : 0;

  if (warp == TMA_WARP) {
    bool ok = true;
    if (n > 0 && lane == 0) {
      mbar_expect_tx(&sh->q_full, (F::KS + F::VS) * rows * 128);
      for (int s = 0; s < F::KS; ++s) tma_rows(sQ + s * SLAB, &tmQ, &sh->q_full, s * 64, head0, q0 + first);
      for (int s = 0; s < F::VS; ++s) tma_rows(sG + s * SLAB, &tmG, &sh->q_full, s * 64, head0, q0 + first);
    }
    for (int j = 0; j < n && ok; ++j) {
      const int ks = j % F::K_SLOTS, vs = j % F::V_SLOTS;
      ok = warp_wait(&sh->k_empty[ks], ((j / F::K_SLOTS) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      const bool cut = (j + 1) * TILE > Lk;                   // K is summed over its rows: those behind the sequence's end become zero
      uint64_t* bar = cut ? &sh->tail : &sh->k_full[ks];
      if (lane == 0) {
        mbar_expect_tx(bar, F::KS * SLAB);
        for (int s = 0; s < F::KS; ++s) tma_rows(sK + (ks * F::KS + s) * SLAB, &tmK, bar, s * 64, kvh, k0 + j * TILE);
      }
      if (cut) {
        ok = warp_wait(bar, 0, abort_flag, a.err, ERR_WAIT_FULL);
        if (!ok) break;
        clear_tail(sK + ks * F::KS * SLAB, F::KS, Lk - j * TILE, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->k_full[ks]);
      }
      ok = warp_wait(&sh->v_empty[vs], ((j / F::V_SLOTS) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&sh->v_full[vs], F::VS * SLAB);
        for (int s = 0; s < F::VS; ++s) tma_rows(sV + (vs * F::VS + s) * SLAB, &tmV, &sh->v_full[vs], s * 64, kvh, k0 + j * TILE);
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------ S = Q K', each half as soon as its compute warps hold the one before ------------------------------
    if (elect_one()) {
      constexpr uint32_t id_s = idesc(HALF, PART, false);
      const uint64_t dK = base_k(smem_u32(sK));
      Ring<F::K_SLOTS> rk;
      bool ok = n == 0 || mbar_wait(&sh->rows_in, 0, abort_flag, a.err, ERR_WAIT_FULL);
      for (int j = 0; j < n && ok; ++j) {
        ok = mbar_wait(&sh->k_full[rk.at], rk.round, abort_flag, a.err, ERR_WAIT_FULL);
        for (int h = 0; h < 2 && ok; ++h) {
          ok = j == 0 || mbar_wait(&sh->s_free[h], (j - 1) & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after();
          const uint64_t d = dK + rk.at * (F::KS * SLAB >> 4) + h * (SLAB / 2 >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) umma_ta(tmem + h * 64, tmem + 384 + k * 8, d + step_k(k), id_s, k != 0);
          umma_commit(&sh->s_full[h]);
        }
        rk.next();
      }
    }
  } else if (warp == MMA_WARP + 1) {
    // ------------------------------ dQ += dS K, then dP = dO V' of the next tile over the columns of dS ------------------------------
    if (elect_one()) {
      constexpr uint32_t id_s = idesc(HALF, PART, false), id_q = idesc(HALF, D, true);
      const uint64_t dK = base_mn(smem_u32(sK)), dV = base_k(smem_u32(sV));
      Ring<F::K_SLOTS> rk;
      Ring<F::V_SLOTS> rv;
      bool ok = n == 0 || mbar_wait(&sh->rows_in, 0, abort_flag, a.err, ERR_WAIT_FULL);
      for (int j = -1; j < n && ok; ++j) {
        if (j >= 0) {
          ok = mbar_wait(&sh->k_full[rk.at], rk.round, abort_flag, a.err, ERR_WAIT_FULL);
          for (int h = 0; h < 2 && ok; ++h) {
            ok = mbar_wait(&sh->ds_full[h], j & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
            const uint64_t d = dK + rk.at * (F::KS * SLAB >> 4) + h * step_mn(4);
#pragma unroll
            for (int k = 0; k < PART / 16; ++k) umma_ta(tmem + 256, tmem + 128 + h * 64 + k * 8, d + step_mn(k), id_q, (j | h | k) != 0);
            umma_commit(&sh->dq_done[h]);
          }
          if (!ok) break;
          umma_commit(&sh->k_empty[rk.at]);
          rk.next();
        }
        if (j + 1 < n) {
          ok = mbar_wait(&sh->v_full[rv.at], rv.round, abort_flag, a.err, ERR_WAIT_FULL);
          for (int h = 0; h < 2 && ok; ++h) {
            ok = j < 0 || mbar_wait(&sh->dq_done[h], j & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
            const uint64_t d = dV + rv.at * (F::VS * SLAB >> 4) + h * (SLAB / 2 >> 4);
#pragma unroll
            for (int k = 0; k < DV / 16; ++k) umma_ta(tmem + 128 + h * 64, tmem + 448 + k * 8, d + step_k(k), id_s, k != 0);
            umma_commit(&sh->dp_full[h]);
          }
          if (ok) umma_commit(&sh->v_empty[rv.at]);
          rv.next();
        }
      }
      if (ok && n > 0) umma_commit(&sh->acc_done);
    }
  } else {
    const int half = warp >> 2, r = tid & 127, tok = r * a.by_hb >> 16, pos = first + tok;
    const bool mine = r < rows && pos < L;
    const int last = mine ? off + pos : -1, head = head0 + (r - tok * a.hb);
    const long long at = (long long)(q0 + pos) * a.heads + head;
    const float delta = mine ? a.delta[at] : 0.f;
    const float lse = (mine ? a.lse[at] : INFINITY) - (HALF ? P_UP : 0.f);
    const uint32_t lane_addr = uint32_t((warp & 3) * 32) << 16;
    bool ok = n == 0 || warp_wait(&sh->q_full, 0, abort_flag, a.err, ERR_WAIT_FULL);
    if (ok && n > 0) {                       // half a row from each of its two threads
      auto fill = [&](const uint8_t* tile, int slabs, uint32_t to) {
        if (half >= slabs) return;
        uint32_t x[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(tile + half * SLAB + r * 128 + ((c ^ (r & 7)) << 4));
          x[c * 4] = v.x; x[c * 4 + 1] = v.y; x[c * 4 + 2] = v.z; x[c * 4 + 3] = v.w;
        }
        tmem_st(to + half * 32 + lane_addr, x);
      };
      fill(sQ, F::KS, tmem + 384);
      fill(sG, F::VS, tmem + 448);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->rows_in);
    }
    float up = 1.f, down = 1.f;              // fp16: of the row's own bound
    if (HALF) {
      powers_for(mine ? a.big[at] * __uint_as_float(a.vtop[(long long)unit.seq * a.kv_heads + kvh]) : 0.f, up, down);
      down *= P_DOWN;
    }
    const float delta_up = delta * up;
    auto tile = [&](int j, auto where) {
      constexpr bool MASK = decltype(where)::value;
      const int lim = last - j * TILE - half * 64;
      const uint32_t tS = tmem + half * 64 + lane_addr, tdP = tmem + 128 + half * 64 + lane_addr;
      if (!warp_wait(&sh->s_full[half], j & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
      float p[64];
      uint32_t s0[32], s1[32];
      tmem_ld_32x32(tS, s0);
      tmem_ld_32x32(tS + 32, s1);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->s_free[half]);
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const uint32_t (&s)[32] = e < 16 ? s0 : s1;
        const float2 x = pr_get(pr_fma(pr(__uint_as_float(s[2 * (e & 15)]), __uint_as_float(s[2 * (e & 15) + 1])), pr(a.scale_log2), pr(-lse)));
        p[2 * e] = !MASK || 2 * e <= lim ? ex2(x.x) : 0.f;
        p[2 * e + 1] = !MASK || 2 * e + 1 <= lim ? ex2(x.y) : 0.f;
      }
      if (!warp_wait(&sh->dp_full[half], j & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
      uint32_t ds[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t d[32];
        tmem_ld_32x32(tdP + c * 32, d);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = c * 32 + 2 * e;
          const Pair dp = pr(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1]));
          const float2 xy = pr_get(pr(p[i], p[i + 1]) * (HALF ? pr_fma(dp, pr(up), pr(-delta_up)) : dp + pr(-delta)));
          float x = xy.x, y = xy.y;
          if (MASK) {                                         // what is not seen may be anything, a NaN too
            x = i <= lim ? x : 0.f;
            y = i + 1 <= lim ? y : 0.f;
          }
          ds[c * 16 + e] = pair<HALF>(x, y);
        }
      }
      tmem_st(tdP, ds);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->ds_full[half]);
      return true;
    };
    for (int j = 0; j < open && ok; ++j) ok = tile(j, Whole{});
    for (int j = open; j < n && ok; ++j) ok = tile(j, Masked{});
    if (ok && n > 0) ok = warp_wait(&sh->acc_done, 0, abort_flag, a.err, ERR_WAIT_TMEM_FULL);
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int col = half * (D / 2) + c * 32;
        uint32_t x[32];
        if (n > 0) {
          tmem_ld_32x32(tmem + 256 + col + lane_addr, x);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = last >= 0 ? __float_as_uint(__uint_as_float(x[e]) * (a.scale * down)) : 0u;
        put_columns<HALF>(sQ, r, col, x);                     // Q is in TMEM
      }
      int places_at[D / 16];
      places(places_at, (warp & 3) * 32, lane, [&](int r) {
        const int tok = r * a.by_hb >> 16;
        return r < rows && first + tok < L ? tok * a.heads + (r - tok * a.hb) : -1;
      });
      send_rows(sQ + (D == 128 ? half * SLAB : 0), (warp & 3) * 32, half * (D / 2), a.dim, lane, places_at,
                reinterpret_cast<uint16_t*>(a.out) + ((long long)(q0 + first) * a.heads + head0) * a.dim);
    }
  }
  tc_fence_before();
  __syncthreads();
  settle(abort_flag);
  if (warp == MMA_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// ---- backward: key and value gradients ---------------------------------------------------------------------------------
template <int D, int DV>
struct Dkv {
  static constexpr int KS = D / 64, VS = DV / 64, STAGES = 2;
  struct Shared {
    uint64_t kv_full, q_full[STAGES], stat_full[STAGES], q_empty[STAGES], tail;
    uint64_t s_full[2], dp_full[2], p_full[2], ds_full[2], dv_done[2], dk_done[2], acc_done;      // half of the query tile
    Unit unit;
    uint32_t tmem_slot;
    int abort_flag;
    alignas(16) float lse[STAGES][TILE], delta[STAGES][TILE];             // their negatives; read four at a time
  };
  static constexpr int SMEM = (1 + STAGES) * (KS + VS) * SLAB + (int)sizeof(Shared) + 1024;
};

template <bool HALF, int D, int DV>
__global__ void __launch_bounds__(THREADS, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmG, const Args a) {
  using F = Dkv<D, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + F::KS * SLAB;
  uint8_t* sQ = sV + F::VS * SLAB;           // stages of Q, then dO
  constexpr int STAGE = (F::KS + F::VS) * SLAB;
  auto* sh = reinterpret_cast<typename F::Shared*>(sQ + F::STAGES * STAGE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int u = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads, group0 = kvh * (a.heads / a.kv_heads);
  const int rows = a.hb * a.tok;
  volatile int* abort_flag = &sh->abort_flag;
  if (warp == 0) {
    const Unit r = find_unit(a, true, TILE, u, lane);
    if (lane == 0) sh->unit = r;
  }
  if (tid == 32) {
    mbar_init(&sh->kv_full, 1);
    for (int s = 0; s < F::STAGES; ++s) {
      mbar_init(&sh->q_full[s], 1);
      mbar_init(&sh->stat_full[s], 1);
      mbar_init(&sh->q_empty[s], 2);
    }
    mbar_init(&sh->tail, 1);
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sh->s_full[h], 1);
      mbar_init(&sh->dp_full[h], 1);
      mbar_init(&sh->p_full[h], 4);
      mbar_init(&sh->ds_full[h], 4);
      mbar_init(&sh->dv_done[h], 1);
      mbar_init(&sh->dk_done[h], 1);
    }
    mbar_init(&sh->acc_done, 2);
    sh->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) { tmem_alloc(&sh->tmem_slot, 512); tmem_relinquish(); }
  if (warp == TMA_WARP && rows < TILE) {     // rows that no copy ever fills are summed too
    for (int s = 0; s < F::STAGES; ++s) clear_tail(sQ + s * STAGE, F::KS + F::VS, rows, lane);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  const bool drain = set_up(a.err);
  tc_fence_after();
  const uint32_t tmem = sh->tmem_slot;       // S' at 0 (P' over it), dP' at 128 (dS' over it), dV at 256, dK at 384
  const Unit unit = sh->unit;
  if (drain || unit.bad || u >= unit.total) {
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
    if (drain) return;
    if (unit.bad) {
      if (tid == 0 && a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
      return;
    }
    clear_rows(a.out, __ldg(a.cu_k + a.n), a.Tk, a.kv_heads, kvh, 1, a.dim, u - unit.total, a.units - unit.total);
    clear_rows(a.out2, __ldg(a.cu_k + a.n), a.Tk, a.kv_heads, kvh, 1, a.vdim, u - unit.total, a.units - unit.total);
    return;
  }
  const int q0 = unit.q0, L = unit.L, k0 = unit.k0, Lk = unit.Lk;
  const int off = Lk - L;
  // place 0 is the last key tile of its sequence, which few queries see: the longest loops come first
  const int kt = (Lk + TILE - 1) / TILE - 1 - unit.place, key0 = kt * TILE;
  const int q_tiles = (L + a.tok - 1) / a.tok, q_first = max(0, key0 - off) / a.tok;
  const int per_chunk = max(0, q_tiles - q_first), n = per_chunk * a.chunks;
  auto tile_of = [&](int i) { return q_tiles - 1 - i % per_chunk; };          // query tile of step i, the last one first
  float up = 1.f, down = 1.f;                // fp16: of the bound of the sequence and key head
  if (HALF) {
    const long long at = (long long)unit.seq * a.kv_heads + kvh;
    powers_for(__uint_as_float(a.top[at]) * __uint_as_float(a.vtop[at]), up, down);
    down *= P_DOWN;
  }

  if (warp == TMA_WARP) {
    bool ok = true;
    if (n > 0 && lane == 0) {
      mbar_expect_tx(&sh->kv_full, (F::KS + F::VS) * SLAB);
      for (int s = 0; s < F::KS; ++s) tma_rows(sK + s * SLAB, &tmK, &sh->kv_full, s * 64, kvh, k0 + key0);
      for (int s = 0; s < F::VS; ++s) tma_rows(sV + s * SLAB, &tmV, &sh->kv_full, s * 64, kvh, k0 + key0);
    }
    uint32_t cuts = 0;
    for (int i = 0; i < n && ok; ++i) {
      const int s = i % F::STAGES, first = tile_of(i) * a.tok, head0 = group0 + i / per_chunk * a.hb;
      ok = warp_wait(&sh->q_empty[s], ((i / F::STAGES) & 1) ^ 1, abort_flag, a.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      const bool cut = first + a.tok > L;                     // Q and dO are summed over their rows
      uint64_t* bar = cut ? &sh->tail : &sh->q_full[s];
      uint8_t* st = sQ + s * STAGE;
      if (lane == 0) {
        mbar_expect_tx(bar, (F::KS + F::VS) * rows * 128);
        for (int c = 0; c < F::KS; ++c) tma_rows(st + c * SLAB, &tmQ, bar, c * 64, head0, q0 + first);
        for (int c = 0; c < F::VS; ++c) tma_rows(st + (F::KS + c) * SLAB, &tmG, bar, c * 64, head0, q0 + first);
      }
      float lse[TILE / 32], delta[TILE / 32];                 // all on their way before the first is put down
#pragma unroll
      for (int c = 0; c < TILE / 32; ++c) {
        const int r = c * 32 + lane, tok = r * a.by_hb >> 16, pos = first + tok;
        const bool mine = r < rows && pos < L;
        const long long at = (long long)(q0 + pos) * a.heads + head0 + (r - tok * a.hb);
        lse[c] = mine ? (HALF ? P_UP : 0.f) - __ldg(a.lse + at) : -INFINITY;
        delta[c] = mine ? __ldg(a.delta + at) * -up : 0.f;
      }
#pragma unroll
      for (int c = 0; c < TILE / 32; ++c) {
        sh->lse[s][c * 32 + lane] = lse[c];
        sh->delta[s][c * 32 + lane] = delta[c];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->stat_full[s]);
      if (cut) {
        ok = warp_wait(bar, cuts & 1, abort_flag, a.err, ERR_WAIT_FULL);
        ++cuts;
        if (!ok) break;
        clear_tail(st, F::KS + F::VS, (L - first) * a.hb, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full[s]);
      }
    }
  } else if (warp >= MMA_WARP) {
    // The first issuing warp: dV += P' dO, then S' = K Q' of the next query tile over the columns of P'; the second: dK += dS' Q, then dP' = V dO'
    // over the columns of dS'.  Half by half, so that the scores of one half are multiplied while the other half is still being used.
    if (elect_one()) {
      const bool second = warp > MMA_WARP;
      constexpr uint32_t id_s = idesc(HALF, PART, false);
      const uint32_t id_g = second ? idesc(HALF, D, true) : idesc(HALF, DV, true), tS = tmem + (second ? 128 : 0), tG = tmem + (second ? 384 : 256);
      const uint32_t q = smem_u32(sQ), g = smem_u32(sQ + F::KS * SLAB);
      const uint64_t dA = base_k(smem_u32(second ? sV : sK)), dB = base_k(second ? g : q), dG = base_mn(second ? q : g);
      uint64_t *scored = second ? sh->dp_full : sh->s_full, *given = second ? sh->ds_full : sh->p_full, *used = second ? sh->dk_done : sh->dv_done;
      const int steps = (second ? DV : D) / 16;
      Ring<F::STAGES> next, now;             // of the scores, of the gradients
      bool ok = n == 0 || mbar_wait(&sh->kv_full, 0, abort_flag, a.err, ERR_WAIT_FULL);
      for (int i = -1; i < n && ok; ++i) {
        if (i >= 0) {
          const uint64_t d = dG + now.at * (STAGE >> 4);
          for (int h = 0; h < 2 && ok; ++h) {
            ok = mbar_wait(&given[h], i & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < PART / 16; ++k) umma_ta(tG, tS + h * 64 + k * 8, d + h * step_mn(4) + step_mn(k), id_g, (i | h | k) != 0);
            umma_commit(&used[h]);
          }
          if (!ok) break;
          umma_commit(&sh->q_empty[now.at]);
          now.next();
        }
        if (i + 1 < n) {
          ok = mbar_wait(&sh->q_full[next.at], next.round, abort_flag, a.err, ERR_WAIT_FULL);
          for (int h = 0; h < 2 && ok; ++h) {
            ok = i < 0 || mbar_wait(&used[h], i & 1, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
            const uint64_t d = dB + next.at * (STAGE >> 4) + h * (SLAB / 2 >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              if (k < steps) umma_f16(tS + h * 64, dA + step_k(k), d + step_k(k), id_s, k != 0);
            umma_commit(&scored[h]);
          }
          next.next();
        }
      }
      if (ok && n > 0) umma_commit(&sh->acc_done);
    }
  } else {
    const int half = warp >> 2, r = tid & 127;
    const uint32_t lane_addr = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + half * 64 + lane_addr, tdP = tmem + 128 + half * 64 + lane_addr;
    auto step = [&](int i, auto where) {
      constexpr bool MASK = decltype(where)::value;
      const int s = i % F::STAGES, first = tile_of(i) * a.tok;
      // columns [from, to) see this key: queries at or behind it, of this sequence
      const int from = max(0, key0 + r - off - first) * a.hb - half * 64, to = min(a.tok, L - first) * a.hb - half * 64;
      if (!warp_wait(&sh->stat_full[s], (i / F::STAGES) & 1, abort_flag, a.err, ERR_WAIT_FULL)) return false;
      if (!warp_wait(&sh->s_full[half], i & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
      float p[64];
      uint32_t w[32];
      uint32_t x0[32], x1[32];
      float4 m[8];
      tmem_ld_32x32(tS, x0);
      tmem_ld_32x32(tS + 32, x1);
      lds_row(m, &sh->lse[s][half * 64]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c == 1) lds_row(m, &sh->lse[s][half * 64 + 32]);
        const uint32_t (&x)[32] = c ? x1 : x0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {                         // lse and delta lie there as they are subtracted
          const float2 u = pr_get(pr_fma(pr(__uint_as_float(x[q * 4]), __uint_as_float(x[q * 4 + 1])), pr(a.scale_log2), pr(m[q].x, m[q].y)));
          const float2 v = pr_get(pr_fma(pr(__uint_as_float(x[q * 4 + 2]), __uint_as_float(x[q * 4 + 3])), pr(a.scale_log2), pr(m[q].z, m[q].w)));
          const float es[4] = {ex2(u.x), ex2(u.y), ex2(v.x), ex2(v.y)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = c * 32 + q * 4 + e;
            p[col] = !MASK || (col >= from && col < to) ? es[e] : 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[c * 16 + e] = pair<HALF>(p[c * 32 + 2 * e], p[c * 32 + 2 * e + 1]);
      }
      tmem_st(tS, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->p_full[half]);
      if (!warp_wait(&sh->dp_full[half], i & 1, abort_flag, a.err, ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t x[32];
        tmem_ld_32x32(tdP + c * 32, x);
        lds_row(m, &sh->delta[s][half * 64 + c * 32]);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int at = c * 32 + q * 4;
          const Pair d0 = pr(__uint_as_float(x[q * 4]), __uint_as_float(x[q * 4 + 1])), d1 = pr(__uint_as_float(x[q * 4 + 2]), __uint_as_float(x[q * 4 + 3]));
          const float2 u = pr_get(pr(p[at], p[at + 1]) * (HALF ? pr_fma(d0, pr(up), pr(m[q].x, m[q].y)) : d0 + pr(m[q].x, m[q].y)));
          const float2 v = pr_get(pr(p[at + 2], p[at + 3]) * (HALF ? pr_fma(d1, pr(up), pr(m[q].z, m[q].w)) : d1 + pr(m[q].z, m[q].w)));
          float d[4] = {u.x, u.y, v.x, v.y};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = at + e;
            if (MASK && !(col >= from && col < to)) d[e] = 0.f;
          }
          w[c * 16 + q * 2] = pair<HALF>(d[0], d[1]);
          w[c * 16 + q * 2 + 1] = pair<HALF>(d[2], d[3]);
        }
      }
      tmem_st(tdP, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->ds_full[half]);
      return true;
    };
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int first = tile_of(i) * a.tok;
      ok = key0 + TILE - 1 > off + first || first + a.tok > L ? step(i, Masked{}) : step(i, Whole{});
    }
    if (ok && n > 0) ok = warp_wait(&sh->acc_done, 0, abort_flag, a.err, ERR_WAIT_TMEM_FULL);
    if (ok) {
      tc_fence_after();
      uint8_t* stage = sQ;                                    // the first stage has been used
#pragma unroll
      for (int c = 0; c < (D + DV) / 64; ++c) {
        const bool k = c < D / 64;
        const int col = k ? half * (D / 2) + c * 32 : half * (DV / 2) + (c - D / 64) * 32;
        uint32_t x[32];
        if (n > 0) {
          tmem_ld_32x32(tmem + (k ? 384 : 256) + col + lane_addr, x);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0u;
        }
        if (k) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * (a.scale * down));
        } else if (HALF) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * P_DOWN);
        }
        put_columns<HALF>(k ? stage : stage + F::KS * SLAB, r, col, x);
      }
      auto place_of = [&](int r) { return key0 + r < Lk ? r * a.kv_heads : -1; };
      const long long first = (long long)(k0 + key0) * a.kv_heads + kvh;
      int k_at[D / 16], v_at[DV / 16];
      places(k_at, (warp & 3) * 32, lane, place_of);
      places(v_at, (warp & 3) * 32, lane, place_of);
      send_rows(stage + (D == 128 ? half * SLAB : 0), (warp & 3) * 32, half * (D / 2), a.dim, lane, k_at, reinterpret_cast<uint16_t*>(a.out) + first * a.dim);
      send_rows(stage + (F::KS + (DV == 128 ? half : 0)) * SLAB, (warp & 3) * 32, half * (DV / 2), a.vdim, lane, v_at,
                reinterpret_cast<uint16_t*>(a.out2) + first * a.vdim);
    }
  }
  tc_fence_before();
  __syncthreads();
  settle(abort_flag);
  if (warp == MMA_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// Calls without rows of queries or of keys: their ends are looked at all the same
__global__ void packed_ends_kernel(const int* cu_q, const int* cu_k, int n, int T, int Tk, int* err) {
  bool bad = false;
  for (int i = threadIdx.x; i <= n; i += blockDim.x) {
    const int x = __ldg(cu_q + i), y = __ldg(cu_k + i);
    bad |= x > T || y > Tk || (i == 0 ? x != 0 || y != 0 : x < __ldg(cu_q + i - 1) || y < __ldg(cu_k + i - 1));
  }
  if (bad && err) atomicCAS(err, 0, ERR_BAD_ARG);
}

// ---- launches --------------------------------------------------------------------------------------------------------
// [rows, heads, width] with strides (elements) of rows and heads; boxes of 64 columns, `box_heads` heads, `box_rows` rows
int map_rows(CUtensorMap* out, const void* base, int rows, int heads, int width, const long long* strides, int box_heads, int box_rows, bool half) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return -1;
  // a stride that no step takes may be anything: one that the encoder accepts stands in its place
  const long long plain = (long long)width * 2;
  cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t st[2] = {(cuuint64_t)(heads > 1 ? strides[1] * 2 : plain), (cuuint64_t)(rows > 1 ? strides[0] * 2 : plain * heads)};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, es[3] = {1, 1, 1};
  const CUresult r = enc(out, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, st, box,
                         es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

static_assert(Fwd<128, 128>::SMEM <= 227 * 1024 && Fwd<128, 64>::SMEM <= 227 * 1024 && Dq<128, 128>::SMEM <= 227 * 1024 &&
                  Dkv<128, 128>::SMEM <= 227 * 1024,
              "shared memory of a block");

template <typename K>
int configure(K kern, int smem, PerDevice& cfg) {
  if (cfg.first()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -2;
    cfg.done();
  }
  return 0;
}

// Tiles of the sequences are at most rows / per + n, since each begins at most one part-filled tile; one block more for the rows behind them
long long units_of(int rows, int n, int per) { return rows / per + (long long)n + 1; }

int shape(Args& a) {
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.dim < 8 || a.dim % 8 || a.dim > 128 || a.vdim < 8 || a.vdim % 8 || a.vdim > 128 ||
      a.T < 1 || a.Tk < 1 || a.n < 0 || !(a.scale >= 0.f) || a.T > (1 << 30) || a.Tk > (1 << 30) || a.n > (1 << 30))
    return -10;
  // Heads of a tile: all of a group where they fill 15/16 of its rows or more, else the largest divisor of the group that does (96 heads: three
  // tiles of 32 heads of 4 tokens rather than one of a single token that leaves a quarter idle).  One head always does.
  const int group = a.heads / a.kv_heads;
  a.hb = group < TILE ? group : TILE;
  while (group % a.hb || TILE / a.hb * a.hb < TILE * 15 / 16) --a.hb;
  a.chunks = group / a.hb;
  a.tok = TILE / a.hb;
  a.by_hb = (65536 + a.hb - 1) / a.hb;       // too large by less than hb / 65536 a step: r hb < 65536
  return 0;
}

// Blocks that share the keys of a pair of query tiles in the forward: as many as there are SMs for, where half of them or more would have nothing to do
// (64 new tokens on 8128 keys, 4 heads over 1: 20 us, 112 unshared; 512 on 7680, 32 heads over 8, two shares: 71 us, 108 unshared).
int splits_of(const Args& a) {
  const long long pairs = (a.T / (2 * a.tok) + (long long)a.n) * a.kv_heads * a.chunks, sms = sm_count() > 0 ? sm_count() : 1;
  const long long most = a.Tk / (FEWEST_TILES * TILE);
  if (pairs < 1 || 2 * pairs > sms || most < 2) return 1;
  return int(sms / pairs < most ? sms / pairs : most);
}

struct Inputs {
  const void *q, *k, *v, *g;
  const long long *qs, *ks, *vs, *gs;
};

int maps(CUtensorMap (&m)[4], const Inputs& i, const Args& a, bool half) {
  int rc = map_rows(&m[0], i.q, a.T, a.heads, a.dim, i.qs, a.hb, a.tok, half);
  if (!rc) rc = map_rows(&m[1], i.k, a.Tk, a.kv_heads, a.dim, i.ks, 1, TILE, half);
  if (!rc) rc = map_rows(&m[2], i.v, a.Tk, a.kv_heads, a.vdim, i.vs, 1, TILE, half);
  if (!rc && i.g) rc = map_rows(&m[3], i.g, a.T, a.heads, a.vdim, i.gs, a.hb, a.tok, half);
  return rc;
}

template <bool HALF, int D, int DV>
int forward(const Inputs& in, Args a, cudaStream_t stream) {
  CUtensorMap m[4];
  int rc = maps(m, in, a, HALF);
  static PerDevice cfg;
  if (!rc) rc = configure(packed_fwd_kernel<HALF, D, DV>, Fwd<D, DV>::SMEM, cfg);
  if (rc) return rc;
  const long long units = units_of(a.T, a.n, 2 * a.tok), pairs = units * a.kv_heads * a.chunks;
  a.splits = a.part ? splits_of(a) : 1;
  if (pairs * a.splits > 0x7fffffffLL) return -10;
  a.units = (int)units;
  packed_fwd_kernel<HALF, D, DV><<<(unsigned)(pairs * a.splits), THREADS, Fwd<D, DV>::SMEM, stream>>>(m[0], m[1], m[2], a);
  if (cudaGetLastError() != cudaSuccess) return -3;
  if (a.splits == 1) return 0;
  return few::launch_early(packed_join_kernel<HALF, DV>, dim3((unsigned)(pairs * 2 * (DV / 8))), dim3(TILE), 0, stream, a);
}

template <bool HALF, int D, int DV>
int backward(const Inputs& in, Args a, void* dq, void* dk, void* dv, cudaStream_t stream) {
  CUtensorMap m[4];
  int rc = maps(m, in, a, HALF);
  static PerDevice cfg_q, cfg_k;
  if (!rc) rc = configure(packed_dq_kernel<HALF, D, DV>, Dq<D, DV>::SMEM, cfg_q);
  if (!rc) rc = configure(packed_dkv_kernel<HALF, D, DV>, Dkv<D, DV>::SMEM, cfg_k);
  if (rc) return rc;
  const long long uq = units_of(a.T, a.n, a.tok), uk = units_of(a.Tk, a.n, TILE);
  if (uq * a.kv_heads * a.chunks > 0x7fffffffLL || uk * a.kv_heads > 0x7fffffffLL) return -10;
  {
    constexpr int LANES = DV / 8, ROWS = DELTA_THREADS / LANES * DELTA_AHEAD;
    const long long blocks = ((long long)a.T * a.heads + ROWS - 1) / ROWS;
    const long long warps = ((long long)(a.T + 31) / 32 + (a.Tk + 31) / 32) * a.kv_heads, sizes = (warps + DELTA_THREADS / 32 - 1) / (DELTA_THREADS / 32);
    if (blocks > 0x7fffffffLL || sizes > 0x7fffffffLL) return -10;
    packed_delta_kernel<HALF, LANES><<<(unsigned)blocks, DELTA_THREADS, 0, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return -3;
    if (HALF) {
      if (cudaMemsetAsync(a.top, 0, 2 * sizeof(uint32_t) * a.n * a.kv_heads, stream) != cudaSuccess) return -3;
      packed_sizes_kernel<LANES><<<(unsigned)sizes, DELTA_THREADS, 0, stream>>>(a);
      if (cudaGetLastError() != cudaSuccess) return -3;
    }
  }
  if (dq) {
    a.units = (int)uq;
    a.out = dq;
    packed_dq_kernel<HALF, D, DV><<<(unsigned)(uq * a.kv_heads * a.chunks), THREADS, Dq<D, DV>::SMEM, stream>>>(m[0], m[1], m[2], m[3], a);
    if (cudaGetLastError() != cudaSuccess) return -3;
  }
  if (!dk) return 0;
  a.units = (int)uk;
  a.out = dk;
  a.out2 = dv;
  packed_dkv_kernel<HALF, D, DV><<<(unsigned)(uk * a.kv_heads), THREADS, Dkv<D, DV>::SMEM, stream>>>(m[0], m[1], m[2], m[3], a);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace
}  // namespace packed
}  // namespace cm

using namespace cm;
using namespace cm::packed;

// Sizes and strides (elements) come in n: strides of tokens and heads of q, k, v (and of go, in the backward); sequences, T, Tk, heads, kv_heads,
// dim, vdim, kind (0 bf16, 1 fp16).  dim, vdim multiples of 8 up to 128; rows on 16 bytes; scale not negative.
static int arguments(Args& a, const int* cu_q, const int* cu_k, float scale, const long long* n, int* err) {
  a.cu_q = cu_q; a.cu_k = cu_k;
  a.n = (int)n[8]; a.T = (int)n[9]; a.Tk = (int)n[10];
  a.heads = (int)n[11]; a.kv_heads = (int)n[12];
  a.dim = (int)n[13]; a.vdim = (int)n[14];
  a.scale = scale; a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err;
  return shape(a);
}

// Floats of work space that the forward wants for these sizes (as below) on the current device; 0: none
extern "C" long long cm_packed_attention_ws(const long long* n) {
  Args a = {};
  if (arguments(a, nullptr, nullptr, 0.f, n, nullptr)) return 0;
  const int splits = splits_of(a);
  return splits == 1 ? 0 : units_of(a.T, a.n, 2 * a.tok) * a.kv_heads * a.chunks * splits * 2 * ((a.vdim > 64 ? 128 : 64) + 3) * TILE;
}

// q [T, heads, dim], k [Tk, kv_heads, dim], v [Tk, kv_heads, vdim]; cu_q, cu_k [sequences + 1]; o [T, heads, vdim] packed; for a backward pass
// o_rest, as o, and lse [T, heads], else null; ws: cm_packed_attention_ws floats, or null
extern "C" int cm_packed_attention_fwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, void* o, void* o_rest,
                                       float* lse, float* ws, const long long* n, float scale, int* err, cudaStream_t stream) {
  Args a = {};
  const int rc = arguments(a, cu_q, cu_k, scale, n, err);
  if (rc) return rc;
  a.out = o;
  a.out2 = o_rest;
  a.lse = lse;
  a.part = ws;
  const Inputs in = {q, k, v, nullptr, n, n + 2, n + 4, nullptr};
  if (n[15] == 0) {
    if (a.vdim > 64) return forward<false, 128, 128>(in, a, stream);
    return a.dim > 64 ? forward<false, 128, 64>(in, a, stream) : forward<false, 64, 64>(in, a, stream);
  }
  if (a.vdim > 64) return forward<true, 128, 128>(in, a, stream);
  return a.dim > 64 ? forward<true, 128, 64>(in, a, stream) : forward<true, 64, 64>(in, a, stream);
}

// o, o_rest and lse from the forward; go (the gradient of o) [T, heads, vdim]; delta: scratch of T * heads floats, fp16: 2 (T heads + sequences kv_heads);
// dq [T, heads, dim], dk [Tk, kv_heads, dim], dv [Tk, kv_heads, vdim] packed, all written whole; dq may be null, or dk and dv together
extern "C" int cm_packed_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_rest, const void* go, const int* cu_q,
                                       const int* cu_k, const float* lse, float* delta, void* dq, void* dk, void* dv, const long long* n, float scale,
                                       int* err, cudaStream_t stream) {
  Args a = {};
  const int rc = arguments(a, cu_q, cu_k, scale, n, err);
  if (rc) return rc;
  a.o = o; a.o_rest = o_rest; a.go = go;
  a.go_tok = n[6]; a.go_head = n[7];
  a.lse = const_cast<float*>(lse);
  a.delta = delta;
  a.big = delta + (long long)a.T * a.heads;
  a.top = reinterpret_cast<uint32_t*>(a.big + (long long)a.T * a.heads);
  a.vtop = a.top + (long long)a.n * a.kv_heads;
  a.v = v; a.v_tok = n[4]; a.v_head = n[5];
  const Inputs in = {q, k, v, go, n, n + 2, n + 4, n + 6};
  if (n[15] == 0) {
    if (a.vdim > 64) return backward<false, 128, 128>(in, a, dq, dk, dv, stream);
    return a.dim > 64 ? backward<false, 128, 64>(in, a, dq, dk, dv, stream) : backward<false, 64, 64>(in, a, dq, dk, dv, stream);
  }
  if (a.vdim > 64) return backward<true, 128, 128>(in, a, dq, dk, dv, stream);
  return a.dim > 64 ? backward<true, 128, 64>(in, a, dq, dk, dv, stream) : backward<true, 64, 64>(in, a, dq, dk, dv, stream);
}

// For T, Tk or heads of zero, where there is nothing to compute: reports ends that do not rise from 0 to at most T and Tk
extern "C" int cm_packed_attention_ends(const int* cu_q, const int* cu_k, long long n, long long T, long long Tk, int* err, cudaStream_t stream) {
  if (n < 0 || T < 0 || Tk < 0 || n >= 1ll << 31 || T >= 1ll << 31 || Tk >= 1ll << 31) return -10;
  packed_ends_kernel<<<1, 256, 0, stream>>>(cu_q, cu_k, (int)n, (int)T, (int)Tk, err);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
