// Rows of bf16, fp16 or fp32 held in registers by a team of TPR threads, VPT packed vectors of N = 16 bytes each.
// VEC: every row starts on a 16-byte boundary and ends on one, and vector i of thread t is the row's vector t + i TPR.  Otherwise rows
// may start and end anywhere: element j of vector i of thread t is the row's element (i N + j) TPR + t, so that neighbouring threads
// move neighbouring elements one at a time (with eight consecutive elements a thread, 16384 x 4095 took 5 times as long as 4096).
// Elements past the row read as zero and are not written.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "fp32_pair.cuh"

namespace cm {

template <typename T>
struct RowVec {
  static constexpr int N = 16 / int(sizeof(T));
  using Bits = uint16_t;
};
template <>
struct RowVec<float> {
  static constexpr int N = 4;
  using Bits = uint32_t;
};

template <typename T>
__device__ __forceinline__ void rv_unpack(const uint4& v, float (&f)[RowVec<T>::N]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  } else {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 p;
      if constexpr (sizeof(T) == 2 && __is_same(T, __half)) p = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
      else p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[j]));
      f[2 * j] = p.x;
      f[2 * j + 1] = p.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 rv_pack(const float (&f)[RowVec<T>::N]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (__is_same(T, __half)) {
        const __half2 p = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        u[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
      }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
}

template <typename T>
__device__ __forceinline__ void rv_unpack(const uint4& v, Pair (&f)[RowVec<T>::N / 2]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < RowVec<T>::N / 2; ++j) {
    if constexpr (sizeof(T) == 4) {
      f[j] = pr(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]));
    } else if constexpr (__is_same(T, __half)) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
      f[j] = pr(p.x, p.y);
    } else {
      f[j] = pr(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 rv_pack(const Pair (&f)[RowVec<T>::N / 2]) {
  float g[RowVec<T>::N];
#pragma unroll
  for (int j = 0; j < RowVec<T>::N / 2; ++j) {
    const float2 p = pr_get(f[j]);
    g[2 * j] = p.x;
    g[2 * j + 1] = p.y;
  }
  return rv_pack<T>(g);
}

// Keeps a vector packed: its unpacked values are formed again after this point instead of being held in registers.
__device__ __forceinline__ void rv_keep_packed(uint4& v) { asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)); }

// a vector of ones
template <typename T>
__device__ __forceinline__ uint4 rv_ones() {
  float f[RowVec<T>::N];
#pragma unroll
  for (int j = 0; j < RowVec<T>::N; ++j) f[j] = 1.f;
  return rv_pack<T>(f);
}

// column of element j of vector i of thread t
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ int rv_column(int t, int i, int j) {
  constexpr int N = RowVec<T>::N;
  return VEC ? (t + i * TPR) * N + j : (i * N + j) * TPR + t;
}

// vector `i` of thread t (zero past the row's end)
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ uint4 rv_load(const T* __restrict__ row, int t, int i, int width) {
  constexpr int N = RowVec<T>::N;
  if constexpr (VEC) {
    return (t + i * TPR) * N < width ? reinterpret_cast<const uint4*>(row)[t + i * TPR] : make_uint4(0, 0, 0, 0);
  } else {
    using Bits = typename RowVec<T>::Bits;
    Bits e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = rv_column<T, TPR, VEC>(t, i, j);
      e[j] = c < width ? reinterpret_cast<const Bits*>(row)[c] : Bits(0);
    }
    if constexpr (sizeof(T) == 4) return make_uint4(e[0], e[1], e[2], e[3]);
    else return make_uint4(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16, e[4] | uint32_t(e[5]) << 16, e[6] | uint32_t(e[7]) << 16);
  }
}

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void rv_store(T* __restrict__ row, int t, int i, int width, const uint4& v) {
  constexpr int N = RowVec<T>::N;
  if constexpr (VEC) {
    if ((t + i * TPR) * N < width) reinterpret_cast<uint4*>(row)[t + i * TPR] = v;
  } else {
    using Bits = typename RowVec<T>::Bits;
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = rv_column<T, TPR, VEC>(t, i, j);
      if (c < width) reinterpret_cast<Bits*>(row)[c] = sizeof(T) == 4 ? Bits(u[j & 3]) : Bits(u[j >> 1] >> ((j & 1) * 16));
    }
  }
}

// Sums of K values over the TPR threads that hold a row, in every one of them.  A team of up to 32 lies within a warp and all lanes
// of the warp take part; a larger one is the whole block.  `red`: [2][K][TPR / 32] floats of shared memory; `turn` alternates
// between calls, so that one barrier a call is enough.
template <int TPR, int K>
__device__ __forceinline__ void rv_team_sum(float (&v)[K], float* red, int turn) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    float* r = red + turn * K * NW;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) r[k * NW + (threadIdx.x >> 5)] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) s += r[k * NW + w];
      v[k] = s;
    }
  }
}

template <int TPR>
constexpr int rv_block() { return TPR < 128 ? 128 : TPR; }

// Column sums that the rows' threads hold, one partial row per block: partial[blockIdx][column].  Teams of the same block are added in
// shared memory (`scratch`, (rows per block) x VPT x TPR x N floats), in a fixed order.
template <typename T, int TPR, int VPT, bool VEC>
__device__ __forceinline__ void rv_partial(const float (&acc)[VPT][RowVec<T>::N], float* __restrict__ out, int width, float* scratch) {
  constexpr int N = RowVec<T>::N, RPB = rv_block<TPR>() / TPR;
  const int t = threadIdx.x % TPR;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = rv_column<T, TPR, VEC>(t, i, j);
        if (c < width) out[c] = acc[i][j];
      }
  } else {
    constexpr int W = VPT * TPR * N;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) scratch[(threadIdx.x / TPR) * W + rv_column<T, TPR, VEC>(t, i, j)] = acc[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += rv_block<TPR>()) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RPB; ++r) s += scratch[r * W + c];
      out[c] = s;
    }
  }
}

template <typename T, int TPR, int VPT, bool VEC>
__device__ __forceinline__ void rv_partial(const Pair (&pairs)[VPT][RowVec<T>::N / 2], float* __restrict__ out, int width, float* scratch) {
  float acc[VPT][RowVec<T>::N];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < RowVec<T>::N / 2; ++j) {
      const float2 p = pr_get(pairs[i][j]);
      acc[i][2 * j] = p.x;
      acc[i][2 * j + 1] = p.y;
    }
  rv_partial<T, TPR, VPT, VEC>(acc, out, width, scratch);
}

// The operand rows of a backward kernel on their way in.  Every thread copies its own vectors of the next NS rows into shared memory
// with asynchronous copies and reads back only what it copied, so the copies need no barrier and keep running over the barriers of the
// rows' sums; read back twice (before and after a row's sum) they take no registers in between.  Rows that
// are not on 16 bytes are loaded when their turn comes and wait in one slot; NS = 0: plain loads, twice.
// What lies past a row's end, past the last row, or belongs to an absent operand is filled with zeros by the copy itself.
template <typename T, int TPR, int VPT, bool VEC, int NS, int OPS>
struct RowRing {
  static constexpr bool ON = VEC && NS > 0, HELD = !VEC && NS > 0;
  static constexpr int TB = rv_block<TPR>(), N = RowVec<T>::N, SLOTS = ON ? NS : 1;
  uint4* mine;               // [ops][NS][VPT][TB], at this thread
  const T* base[OPS];        // first row; null: zero
  long long pitch[OPS];
  int ops, width, first;     // first: this thread's first vector
  long long rows, row, ahead, step;
  int slot;

  __device__ __forceinline__ void set(int op, const void* p, long long elements) {
    base[op] = reinterpret_cast<const T*>(p);
    pitch[op] = elements;
  }
  // the copies of the row NS rows ahead, into the slot that has just been used
  __device__ __forceinline__ void request() {
    if constexpr (ON) {
      const bool there = ahead < rows;
#pragma unroll
      for (int op = 0; op < OPS; ++op) {
        if (op < ops) {
          const T* src = base[op] ? base[op] + ahead * pitch[op] + first * N : nullptr;
#pragma unroll
          for (int i = 0; i < VPT; ++i) {
            const bool on = src && there && (first + i * TPR) * N < width;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(mine + (op * SLOTS * VPT + i) * TB + slot * (VPT * TB))),
                         "l"(on ? src + i * (TPR * N) : base[0]), "r"(on ? 16 : 0)
                         : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      slot = slot + 1 == SLOTS ? 0 : slot + 1;
    }
    ahead += step;
  }
  __device__ __forceinline__ void start(uint4* shared, long long first_row, long long rows_apart) {
    mine = shared + threadIdx.x;
    first = int(threadIdx.x) % TPR;
    row = ahead = first_row;
    step = rows_apart;
    slot = 0;
    if constexpr (ON)
      for (int s = 0; s < NS; ++s) request();
  }
  __device__ __forceinline__ uint4 fetch(int op, int i) const {
    return rv_load<T, TPR, VEC>(base[op] + row * pitch[op], first, i, base[op] && row < rows ? width : 0);
  }
  __device__ __forceinline__ void wait() {
    if constexpr (ON) asm volatile("cp.async.wait_group %0;" ::"n"(NS > 0 ? NS - 1 : 0) : "memory");
    if constexpr (HELD) {
#pragma unroll
      for (int op = 0; op < OPS; ++op) {
        if (op < ops) {
#pragma unroll
          for (int i = 0; i < VPT; ++i) mine[(op * VPT + i) * TB] = fetch(op, i);
        }
      }
    }
  }
  __device__ __forceinline__ uint4 get(int op, int i) const {
    if constexpr (ON || HELD) return mine[(op * SLOTS * VPT + i) * TB + slot * (VPT * TB)];
    else return fetch(op, i);
  }
  // no copy may be on its way when the block ends
  __device__ __forceinline__ void drain() {
    if constexpr (ON) asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // this row has been read
  __device__ __forceinline__ void next() {
    request();
    row += step;
  }
};

// Rows ahead of a backward kernel, by the vectors that a block holds of one operand.
constexpr int rv_stages(int tpr, int vpt) {
  const int held = (tpr < 128 ? 128 : tpr) * vpt;
  return held <= 256 ? 4 : held <= 512 ? 3 : held <= 1024 ? 2 : 0;
}
// Slots of shared memory for one operand.
constexpr int rv_slots(int tpr, int vpt, bool vec) { return vec ? rv_stages(tpr, vpt) : rv_stages(tpr, vpt) > 0 ? 1 : 0; }

// Blocks of a backward kernel: those that the SMs hold at once, up to this many for each, shared by `share` sections of the rows; and no
// more than there are rows.  (Four blocks of 128 threads an SM left the gated norm's backward waiting for memory: 281 us, 16 warps.)
static inline long long rv_most_blocks(long long rows, int width, int share) {
  const int per_sm = width / share <= 2048 ? 8 : 4;
  const long long most = ((long long)sm_count() * per_sm + share - 1) / share;
  return rows < most ? rows : most;
}
// Blocks of one kernel, with one amount of shared memory, that an SM holds: the runtime's answer, kept per device.  Backward passes on
// several devices ask from several host threads.
struct Resident {
  std::atomic<int> kept[64] = {};
  template <typename K>
  int blocks(K kern, int threads, int smem) {
    int dev = -1, n = 0;
    const bool keep = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    if (keep && (n = kept[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) != cudaSuccess || n < 1) return 1;
    if (keep) kept[dev].store(n, std::memory_order_relaxed);
    return n;
  }
};
template <typename K>
static int rv_blocks(K kern, int threads, int smem, int rows_per_block, long long rows, int width, int share, Resident& resident) {
  const long long want = (rows + rows_per_block - 1) / rows_per_block;
  const long long fit = ((long long)sm_count() * resident.blocks(kern, threads, smem) + share - 1) / share;
  const long long most = rv_most_blocks(rows, width, share), n = fit < most ? fit : most;
  return int(want < n ? want : n);
}

// out[c] = sum over p of partial[p][c], c < width, in a fixed order; blockIdx.y chooses one of up to three sums.  32 threads share a
// column: with 8, and one load in flight each, 592 partial rows of 4096 took 16 us.
struct ColumnSums {
  const float* partial[3];
  void* out[3];
};

template <typename T>
__global__ void __launch_bounds__(1024) rv_column_sum(const ColumnSums s, int parts, int width) {
  __shared__ float red[32][33];
  const float* __restrict__ in = s.partial[blockIdx.y];
  T* out = reinterpret_cast<T*>(s.out[blockIdx.y]);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int p = w; p < parts; p += 32) a += in[(long long)p * width + c];
  }
  red[w][lane] = a;
  __syncthreads();
  const float t = warp_sum(red[lane][w]);
  if (lane == 0 && blockIdx.x * 32 + w < width) out[blockIdx.x * 32 + w] = T(t);
}

enum RowType : int { ROW_BF16 = 0, ROW_FP16 = 1, ROW_FP32 = 2 };

// The team of a row of `nvec` vectors, as 16 * threads + vectors a thread; 0: too wide.  `by_warp`: up to 128 vectors go to one warp.
static inline int rv_team(int nvec, bool vec, bool by_warp) {
  if (vec && by_warp && nvec > 64 && nvec <= 128) return 16 * 32 + 4;
  return nvec <= 8 ? 16 * 8 + 1 : nvec <= 32 ? 16 * 32 + 1 : nvec <= 64 ? 16 * 32 + 2 : nvec <= 128 ? 16 * 128 + 1
         : nvec <= 256 ? 16 * 128 + 2 : nvec <= 512 ? 16 * 256 + 2 : nvec <= 1024 ? 16 * 512 + 2 : nvec <= 2048 ? 16 * 1024 + 2
         : nvec <= 4096 ? 16 * 1024 + 4 : 0;
}

// CM_ROW_TEAM(team, vec, F): calls F(threads, vectors, vec) with compile-time values; -10 for a team that does not exist.  Rows have up to
// 16384 elements of type T: the largest team is one of 32-bit rows.
#define CM_ROW_TEAMS(team, VEC, F)                     \
  switch (team) {                                      \
    case 16 * 8 + 1: return F(8, 1, VEC);              \
    case 16 * 32 + 1: return F(32, 1, VEC);            \
    case 16 * 32 + 2: return F(32, 2, VEC);            \
    case 16 * 128 + 1: return F(128, 1, VEC);          \
    case 16 * 128 + 2: return F(128, 2, VEC);          \
    case 16 * 256 + 2: return F(256, 2, VEC);          \
    case 16 * 512 + 2: return F(512, 2, VEC);          \
    case 16 * 1024 + 2: return F(1024, 2, VEC);        \
    case 16 * 1024 + 4:                                \
      if constexpr (sizeof(T) == 4) return F(1024, 4, VEC); \
      break;                                           \
  }
#define CM_ROW_TEAM(team, vec, F)                      \
  if (vec) {                                           \
    CM_ROW_TEAM_BY_WARP(team, F)                       \
    CM_ROW_TEAMS(team, true, F)                        \
  } else {                                             \
    CM_ROW_TEAMS(team, false, F)                       \
  }                                                    \
  return -10

}  // namespace cm
