// Rows of a paged key-value cache: written (quantised on the way where the cache holds E4M3) and read back into packed sequences.
//
//   write   cache[slot / page, slot % page, h, :] = x[t, h, :]               16-bit caches: the same bits
//           e4m3(x / 2^e), e = ceil(log2(max |x| / 448))                     E4M3 caches, one exponent byte e + 127 per row (token, head)
//   read    y[t, h, :] = cache[table[s, p / page], p % page, h, :] (x 2^e)   t the p-th token of sequence s
//
// One power of two per row: multiplying by it is exact, so a value is rounded once, to the 4 bits of E4M3, and the attention that reads the
// cache can leave the power out of its products.  The exponent's largest value is taken over the finite values of the row; what is not finite is
// stored as NaN.
//
// Both are copies: bytes in and out at the memory's rate is all there is.  A row belongs to 8 or 16 lanes, 16 bytes of it to each (8 of an
// E4M3 row), so rows of any stride move in whole sectors, and four rows of every lane group are in flight at once.  Measured: 4095 tokens of 32
// heads, 128 + 64 wide in bf16: write 22 us, read 16 (15 each at the copy rate, though much of it stays in L2); 16384 tokens of 8 heads, 128 + 128 into
// E4M3: write 26 us of 16 (issue slots: a row's maximum, its exponent, four instructions a pair of values), back 20 of 16.
//
// Of tokens that are given the same slot the last one stays, whatever order the blocks run in: each block looks for its own slots among the
// later tokens (a hash table of its own in shared memory, slots of one place in a chain).  It reads the list of slots once per block: 4 us of the
// 26 at 16384 tokens of 8 heads, 10 of 98 at 65536.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "fp32_pair.cuh"
#include "paged.cuh"

namespace cm {
namespace paged {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 128;              // tokens of one block
constexpr int TABLE = 2048;                  // places of the hash table
constexpr int NONE = -1;                     // a place that no slot falls to, the end of a chain
constexpr int ROWS_AHEAD = 4;
constexpr int SCAN = 8;                      // later slots that a thread has on their way at once

// r / n for r < 128 n: by a product where that is exact (r n < 2^32), by a division else
struct Divide {
  uint32_t n, magic;
  __host__ Divide(int heads = 1) : n(heads), magic(heads > 1 && heads < 5000 ? uint32_t(((1ull << 32) + heads - 1) / heads) : 0) {}
  __device__ __forceinline__ int operator()(int r) const { return n == 1 ? r : magic ? int(__umulhi(uint32_t(r), magic)) : int(uint32_t(r) / n); }
};

struct Side {                                // keys or values
  const uint8_t* x;                          // rows of the packed tensor
  uint8_t* cache;
  uint8_t* scale;                            // [pages, page, heads] or null
  long long c_page;                          // strides in bytes
  int x_tok, x_head, c_tok, c_head;
  int lanes, width;                          // lanes of a row (8, 16 or 32), 16-byte pieces of the packed row (8 values each)
  int wide;                                  // an E4M3 cache whose rows are whole 16-byte pieces
};

__device__ __forceinline__ uint32_t place_of(long long slot) { return (uint32_t(slot) * 2654435769u) >> 21; }
static_assert(TABLE == 1 << 11, "place_of");

struct WriteArgs {
  Side side[2];
  int sides;
  const void* slots;
  long long total;                           // slots of the cache
  int wide;                                  // slots are 64-bit
  int T, heads, page, per_block;
  Divide by_heads;
  int* err;
};

__device__ __forceinline__ long long slot_of(const WriteArgs& a, long long t) {
  return a.wide ? reinterpret_cast<const long long*>(a.slots)[t] : (long long)reinterpret_cast<const int*>(a.slots)[t];
}

template <typename T>
__device__ __forceinline__ float2 two(uint32_t v);
template <>
__device__ __forceinline__ float2 two<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 two<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t join(float a, float b);
template <>
__device__ __forceinline__ uint32_t join<__nv_bfloat16>(float a, float b) { return pack_bf16(a, b); }
template <>
__device__ __forceinline__ uint32_t join<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// exponent byte of a row's largest magnitude: the smallest e with amax <= 448 * 2^e = 1.75 * 2^(e + 8), read off its bits
__device__ __forceinline__ int exponent_byte(float amax) {
  if (!(amax > 0.f)) return 127;
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return e < 1 ? 1 : e;                      // at most 254 - 8 + 1
}

// eight values times a power of two as E4M3; infinities and NaN (which a warp's rows have or have not) become NaN
template <typename T, bool FINITE>
__device__ __forceinline__ uint2 quantised(const uint4& v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t out[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = two<T>(w[i]);
    uint32_t b = __nv_cvt_float2_to_fp8x2(pr_get(pr(f.x, f.y) * pr(inv)), __NV_SATFINITE, __NV_E4M3);
    if (!FINITE) {
      if (!isfinite(f.x)) b = (b & 0xff00u) | 0x7fu;
      if (!isfinite(f.y)) b = (b & 0x00ffu) | 0x7f00u;
    }
    out[i >> 1] |= b << (16 * (i & 1));
  }
  return make_uint2(out[0], out[1]);
}

// Magnitudes of 16-bit floats order as their bits do without the sign: the largest of eight, two to an instruction
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t largest_bits(const uint4& v) {
  const uint32_t m = 0x7fff7fffu;
  return max2(max2(v.x & m, v.y & m), max2(v.z & m, v.w & m));
}
template <typename T>
constexpr uint32_t first_not_finite() { return std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u; }

template <typename T>
__device__ float largest_finite(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = two<T>(w[i]);
    if (isfinite(f.x)) m = fmaxf(m, fabsf(f.x));
    if (isfinite(f.y)) m = fmaxf(m, fabsf(f.y));
  }
  return m;
}

// T: the packed rows' type; E4M3: what the cache holds (the same type otherwise); LANES: of a row; PIECES: of 16 bytes to a lane.  The block's tokens
// of one side.  Two pieces a lane where rows are quantised and lie on 16 bytes: what is done once per lane (the row's place, its largest value,
// its exponent) then serves 16 values, and 16 bytes are stored at once.
template <typename T, bool E4M3, int LANES, int PIECES>
__device__ __forceinline__ void write_rows(const Side& d, const Divide& by_heads, int heads, int n, long long t0, const long long* own, const int* lost,
                                           const long long* base) {
  constexpr int GROUPS = THREADS / LANES, AHEAD = ROWS_AHEAD / PIECES;
  const int group = threadIdx.x / LANES, part = threadIdx.x % LANES, rows = n * heads;
  const uint8_t* x = d.x + t0 * d.x_tok + part * PIECES * 16;
  uint8_t* cache = d.cache + part * PIECES * (E4M3 ? 8 : 16);
  const bool exists = part * PIECES < d.width;
  // whole rounds, so that the lanes of a warp meet in the shuffles
  for (int r0 = group; r0 - group < rows; r0 += GROUPS * AHEAD) {
    uint4 v[AHEAD][PIECES];
    int tok[AHEAD], head[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int r = r0 + u * GROUPS;
      tok[u] = by_heads(r);
      head[u] = r - tok[u] * heads;
      if (r >= rows || own[tok[u]] < 0 || lost[tok[u]]) tok[u] = -1;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) v[u][i] = make_uint4(0, 0, 0, 0);
      if (tok[u] >= 0 && exists) {
        const uint4* src = reinterpret_cast<const uint4*>(x + (long long)tok[u] * d.x_tok + (long long)head[u] * d.x_head);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) v[u][i] = __ldg(src + i);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      uint8_t* row = cache + base[tok[u] < 0 ? 0 : tok[u]] + (long long)head[u] * d.c_head;
      if (!E4M3) {
        if (tok[u] >= 0 && exists) *reinterpret_cast<uint4*>(row) = v[u][0];
        continue;
      }
      uint32_t most = largest_bits(v[u][0]);
      if (PIECES == 2) most = max2(most, largest_bits(v[u][PIECES - 1]));
#pragma unroll
      for (int o = LANES >> 1; o > 0; o >>= 1) most = max2(most, __shfl_xor_sync(0xffffffffu, most, o));
      most = max(most & 0xffffu, most >> 16);
      const bool finite = __all_sync(0xffffffffu, most < first_not_finite<T>());             // all values of the warp's rows
      float m = two<T>(most).x;
      if (!finite) {                                          // the row's largest finite one
        m = largest_finite<T>(v[u][0]);
        if (PIECES == 2) m = fmaxf(m, largest_finite<T>(v[u][PIECES - 1]));
#pragma unroll
        for (int o = LANES >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      if (tok[u] < 0) continue;
      const int e = exponent_byte(m);
      if (exists) {
        const float inv = __uint_as_float((254u - e) << 23);  // 2^(127 - e): a subnormal for e = 254 alone, which exponent_byte does not reach
        const uint2 y = finite ? quantised<T, true>(v[u][0], inv) : quantised<T, false>(v[u][0], inv);
        if (PIECES == 2) {
          const uint4& w = v[u][PIECES - 1];
          const uint2 z = finite ? quantised<T, true>(w, inv) : quantised<T, false>(w, inv);
          *reinterpret_cast<uint4*>(row) = make_uint4(y.x, y.y, z.x, z.y);
        } else {
          *reinterpret_cast<uint2*>(row) = y;
        }
      }
      if (part == 0) d.scale[own[tok[u]] * heads + head[u]] = (uint8_t)e;
    }
  }
}

template <typename T, bool E4M3>
__global__ void __launch_bounds__(THREADS, 4) cache_write_kernel(const WriteArgs a) {
  __shared__ int table[TABLE];               // hash place -> a token of this block
  __shared__ int next[MAX_TOKENS];           // -> another one whose slot falls to the same place
  __shared__ long long own[MAX_TOKENS];      // the slot, or -1: not written
  __shared__ long long base[2][MAX_TOKENS];  // and where it begins in the caches
  __shared__ int lost[MAX_TOKENS];           // a later token has the same slot
  const long long t0 = (long long)blockIdx.x * a.per_block;
  const int n = (int)min((long long)a.per_block, a.T - t0);
  for (int i = threadIdx.x; i < TABLE; i += THREADS) table[i] = NONE;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    long long s = slot_of(a, t0 + i);
    if (s >= a.total) {
      if (a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
      s = -1;
    }
    own[i] = s < 0 ? -1 : s;
    lost[i] = 0;
    if (s >= 0) {
      next[i] = atomicExch(&table[place_of(s)], i);
      const long long page = s / a.page, in = s - page * a.page;
      for (int w = 0; w < a.sides; ++w) base[w][i] = page * a.side[w].c_page + in * a.side[w].c_tok;
    }
  }
  __syncthreads();
  for (long long t = t0 + 1 + threadIdx.x; t < a.T; t += SCAN * THREADS) {
    long long s[SCAN];
#pragma unroll
    for (int c = 0; c < SCAN; ++c) s[c] = t + c * THREADS < a.T ? slot_of(a, t + c * THREADS) : -1;
#pragma unroll
    for (int c = 0; c < SCAN; ++c) {
      const int before = (int)min((long long)n, t + c * THREADS - t0);
      for (int at = s[c] < 0 ? NONE : table[place_of(s[c])]; at != NONE; at = next[at])
        if (at < before && own[at] == s[c]) lost[at] = 1;
    }
  }
  __syncthreads();
  for (int w = 0; w < a.sides; ++w) {
    const Side& d = a.side[w];
    if (E4M3 && d.wide && d.width <= 16) write_rows<T, E4M3, 8, 2>(d, a.by_heads, a.heads, n, t0, own, lost, base[w]);
    else if (d.lanes == 8) write_rows<T, E4M3, 8, 1>(d, a.by_heads, a.heads, n, t0, own, lost, base[w]);
    else if (d.lanes == 16) write_rows<T, E4M3, 16, 1>(d, a.by_heads, a.heads, n, t0, own, lost, base[w]);
    else write_rows<T, E4M3, 32, 1>(d, a.by_heads, a.heads, n, t0, own, lost, base[w]);
  }
}

struct ReadArgs {
  Side side[2];                              // x: the packed rows that are written
  int sides;
  const int* table;
  long long table_row;                       // elements between the table's rows
  const int* ends;                           // [sequences + 1]
  int sequences, columns, pages;
  int T, heads, page, per_block;
  Divide by_heads;
  int* err;
};

// eight E4M3 values (x, y) times the power of their exponent byte (z)
template <typename T>
__device__ __forceinline__ uint4 expanded(const uint4& v) {
  const float scale = power_of(v.z);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((i < 2 ? v.x : v.y) >> (16 * (i & 1))), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    o[i] = join<T>(f.x * scale, f.y * scale);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T, bool E4M3, int LANES>
__device__ __forceinline__ void read_rows(const Side& d, const Divide& by_heads, int heads, int n, long long t0, const long long* own,
                                          const long long* base) {
  constexpr int GROUPS = THREADS / LANES;
  const int group = threadIdx.x / LANES, part = threadIdx.x % LANES, rows = n * heads;
  if (part >= d.width) return;
  uint8_t* x = const_cast<uint8_t*>(d.x) + t0 * d.x_tok + part * 16;
  const uint8_t* cache = d.cache + part * (E4M3 ? 8 : 16);
  for (int r0 = group; r0 < rows; r0 += GROUPS * ROWS_AHEAD) {
    uint4 v[ROWS_AHEAD];                     // of an E4M3 row: eight values and its exponent byte
    int tok[ROWS_AHEAD], head[ROWS_AHEAD];
#pragma unroll
    for (int u = 0; u < ROWS_AHEAD; ++u) {
      const int r = r0 + u * GROUPS;
      v[u] = make_uint4(0, 0, 127, 0);
      if (!E4M3) v[u].z = 0;
      tok[u] = by_heads(r);
      head[u] = r - tok[u] * heads;
      if (r >= rows || own[tok[u]] < 0) continue;
      const uint8_t* row = cache + base[tok[u]] + (long long)head[u] * d.c_head;
      if (E4M3) {
        const uint2 b = __ldg(reinterpret_cast<const uint2*>(row));
        v[u].x = b.x;
        v[u].y = b.y;
        v[u].z = __ldg(d.scale + own[tok[u]] * heads + head[u]);
      } else {
        v[u] = __ldg(reinterpret_cast<const uint4*>(row));
      }
    }
#pragma unroll
    for (int u = 0; u < ROWS_AHEAD; ++u) {
      if (r0 + u * GROUPS >= rows) continue;
      *reinterpret_cast<uint4*>(x + (long long)tok[u] * d.x_tok + (long long)head[u] * d.x_head) = E4M3 ? expanded<T>(v[u]) : v[u];
    }
  }
}

template <typename T, bool E4M3>
__global__ void __launch_bounds__(THREADS, 6) cache_read_kernel(const ReadArgs a) {
  __shared__ long long own[MAX_TOKENS];      // page * (slots of a page) + place, or -1: a row of zeros
  __shared__ long long base[2][MAX_TOKENS];  // and where it begins in the caches
  const long long t0 = (long long)blockIdx.x * a.per_block;
  const int n = (int)min((long long)a.per_block, a.T - t0);
  if (blockIdx.x == 0)                       // ends that do not rise from 0 to at most T are reported; no row comes from outside the cache for them
    for (int i = threadIdx.x; i <= a.sequences; i += THREADS) {
      const int end = __ldg(a.ends + i);
      if ((i == 0 ? end != 0 : end < __ldg(a.ends + i - 1)) || end > a.T)
        if (a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
    }
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int t = (int)t0 + i;
    int lo = 0, hi = a.sequences;            // the last sequence that begins at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.ends + mid) <= t) lo = mid;
      else hi = mid;
    }
    int page = -1, at = 0;
    const int begin = a.sequences > 0 ? __ldg(a.ends + lo) : 0;
    if (a.sequences > 0 && begin >= 0 && begin <= t && t < __ldg(a.ends + lo + 1)) {
      const int pos = t - begin, col = pos / a.page;
      at = pos - col * a.page;
      page = col < a.columns ? __ldg(a.table + lo * a.table_row + col) : -1;
      if (page < 0 || page >= a.pages) {
        page = -1;
        if (a.err) atomicCAS(a.err, 0, ERR_BAD_ARG);
      }
    }
    own[i] = page < 0 ? -1 : (long long)page * a.page + at;
    for (int w = 0; w < a.sides; ++w) base[w][i] = page * a.side[w].c_page + (long long)at * a.side[w].c_tok;
  }
  __syncthreads();
  for (int w = 0; w < a.sides; ++w) {
    const Side& d = a.side[w];
    if (d.lanes == 8) read_rows<T, E4M3, 8>(d, a.by_heads, a.heads, n, t0, own, base[w]);
    else if (d.lanes == 16) read_rows<T, E4M3, 16>(d, a.by_heads, a.heads, n, t0, own, base[w]);
    else read_rows<T, E4M3, 32>(d, a.by_heads, a.heads, n, t0, own, base[w]);
  }
}

// Tokens of one block: enough blocks for `resident` on every SM, and then as many tokens as the block's tables hold
static int tokens_per_block(int T, int resident) {
  const int sms = sm_count() > 0 ? sm_count() : 1;
  const int n = (T + resident * sms - 1) / (resident * sms);
  return n < 1 ? 1 : n > MAX_TOKENS ? MAX_TOKENS : n;
}

static Side side_of(const void* x, const long long* xs, void* cache, const long long* cs, void* scale, int width, int esize) {
  Side d;
  d.x = (const uint8_t*)x;
  d.x_tok = int(xs[0] * 2);
  d.x_head = int(xs[1] * 2);
  d.cache = (uint8_t*)cache;
  d.c_page = cs[0] * esize;
  d.c_tok = int(cs[1] * esize);
  d.c_head = int(cs[2] * esize);
  d.scale = (uint8_t*)scale;
  d.width = width / 8;
  d.wide = esize == 1 && width % 16 == 0 && ((reinterpret_cast<uintptr_t>(cache) | d.c_page | d.c_tok | d.c_head) & 15) == 0;
  d.lanes = d.width <= 8 ? 8 : d.width <= 16 ? 16 : 32;
  return d;
}

template <typename A, typename Kern>
static int start(Kern kern, A& a, int resident, cudaStream_t stream) {
  a.per_block = tokens_per_block(a.T, resident);
  const int blocks = (a.T + a.per_block - 1) / a.per_block;
  kern<<<blocks > 0 ? blocks : 1, THREADS, 0, stream>>>(a);   // of no tokens and of no heads what is given is looked at all the same
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace paged
}  // namespace cm

using namespace cm;
using namespace cm::paged;

// Sizes and strides come in one array of 64-bit numbers, strides in elements:
//   k_tok, k_head, v_tok, v_head of the packed rows; page, token and head strides of the key cache, then of the value cache;
//   T, heads, dim, vdim (0: no values), pages, page, kind (0 bf16, 1 fp16), e4m3, then what the function says.
// Packed rows k [T, heads, dim], v [T, heads, vdim]; caches [pages, page, heads, .]; with e4m3 the caches hold E4M3 and k_scale, v_scale
// [pages, page, heads] their exponent bytes.  Widths are multiples of 8 up to 256; rows on 16 bytes (8 in an E4M3 cache); all strides but
// those of pages below 2^31 bytes.
template <typename A>
static int common(A& a, void* k, void* v, void* kc, void* vc, void* k_scale, void* v_scale, const long long* n) {
  const int es = n[17] ? 1 : 2, dim = (int)n[12], vdim = (int)n[13];
  if (dim < 8 || dim % 8 || dim > 256 || vdim < 0 || vdim % 8 || vdim > 256 || n[15] < 1 || n[14] < 0) return -10;
  if (n[17] && n[11] && n[14] && (!k_scale || (vdim && !v_scale))) return -10;             // a cache of nothing may lie nowhere
  for (int i : {0, 1, 2, 3, 5, 6, 8, 9})
    if (n[i] < -(1ll << 30) || n[i] >= 1ll << 30) return -10;
  a.side[0] = side_of(k, n, kc, n + 4, k_scale, dim, es);
  a.sides = 1;
  if (vdim) a.side[a.sides++] = side_of(v, n + 2, vc, n + 7, v_scale, vdim, es);
  a.T = (int)n[10];
  a.heads = (int)n[11];
  a.by_heads = Divide(a.heads);
  a.page = (int)n[15];
  return 0;
}

// Then: slots are 64-bit numbers.  slots [T]: page * (slots of a page) + offset, negative: left out.
extern "C" int cm_cache_write(const void* k, const void* v, void* kc, void* vc, void* k_scale, void* v_scale, const void* slots, const long long* n,
                              int* err, cudaStream_t stream) {
  if (n[10] == 0) return 0;
  if (n[10] < 0 || n[11] < 0) return -10;
  WriteArgs a;
  const int rc = common(a, const_cast<void*>(k), const_cast<void*>(v), kc, vc, k_scale, v_scale, n);
  if (rc) return rc;
  a.slots = slots;
  a.wide = (int)n[18];
  a.total = n[14] * n[15];
  a.err = err;
  if (n[16] == 0) return n[17] ? start(cache_write_kernel<__nv_bfloat16, true>, a, 4, stream) : start(cache_write_kernel<__nv_bfloat16, false>, a, 4, stream);
  return n[17] ? start(cache_write_kernel<__half, true>, a, 4, stream) : start(cache_write_kernel<__half, false>, a, 4, stream);
}

// Then: elements between the rows of the table, sequences, columns of the table.  Token t of the packed results is the (t - ends[s])-th of the
// sequence s that holds it; tokens of no sequence become zeros.
extern "C" int cm_cache_read(void* k, void* v, const void* kc, const void* vc, const void* k_scale, const void* v_scale, const int* table,
                             const int* ends, const long long* n, int* err, cudaStream_t stream) {
  if (n[10] < 0 || n[11] < 0) return -10;
  ReadArgs a;
  const int rc = common(a, k, v, const_cast<void*>(kc), const_cast<void*>(vc), const_cast<void*>(k_scale), const_cast<void*>(v_scale), n);
  if (rc) return rc;
  a.table = table;
  a.table_row = n[18];
  a.ends = ends;
  a.sequences = (int)n[19];
  a.columns = (int)n[20];
  a.pages = (int)n[14];
  a.err = err;
  if (n[16] == 0) return n[17] ? start(cache_read_kernel<__nv_bfloat16, true>, a, 8, stream) : start(cache_read_kernel<__nv_bfloat16, false>, a, 8, stream);
  return n[17] ? start(cache_read_kernel<__half, true>, a, 8, stream) : start(cache_read_kernel<__half, false>, a, 8, stream);
}
