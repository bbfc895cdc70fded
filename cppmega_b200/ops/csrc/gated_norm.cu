// Gated RMS norm of a mixer's output, forward and backward, in bf16, fp16 or fp32.  Groups of `group` channels normalise apart
// (rms(v) = v * rsqrt(mean(v^2) + eps)), a(z) = z sigmoid(z):
//   norm first:  y = rms(x) w a(z)          gate first:  y = rms(x a(z)) w          without z: y = rms(x) w
// Backward, with xh the normalised values, r the reciprocal norm and dn = dy a(z) (norm first) or dy:
//   du = r (dn w - xh mean(dn w xh));  dw = sum dn xh
//   norm first:  dx = du,  dz = dy xh w a'(z)         gate first:  dx = du a(z),  dz = du x a'(z)
// A team of threads holds one group of one row; blockIdx.y is the group, so that a thread keeps its channels over the rows of the
// backward and adds their weight gradient in registers.  Bound by memory: three rows moved forward, five backward (16384 x 8192 in groups of
// 1024, bf16: 134 us and 219, at the copy rate 125 and 208; with the gate first 139 and 280); the gate is read
// where it lies (a column slice of the projection has its own pitch).  The weight gradient is summed in a fixed order.
#include "row_vec.cuh"
#define CM_ROW_TEAM_BY_WARP(team, F) if (team == 16 * 32 + 4) return F(32, 4, true);

namespace cm {

// sigmoid(z).  fp32 rows: z log2(e) in two parts, t and what its rounding and log2(e)'s left out, 2^(t + r) = 2^t (1 + r ln 2): with t alone the
// result errs by |z| 2^-24, at z = -80 sixty times more than by the other steps.  16-bit results round at 2^-12 and more, and t is enough.
// |z| above 104 changes nothing in fp32, and is kept out of the products.  Rows on 16 bytes take as long as with t alone (16384 x 8192 in groups
// of 1024, fp32: 237 us forward, 446 backward), others up to a quarter longer (16384 x 5 groups of 333: 85 for 69 and 134 for 123).
template <typename T>
__device__ __forceinline__ float gate_sigmoid(float z) {
  if constexpr (sizeof(T) == 4) {
    constexpr float L = 1.44269502f, L_REST = 1.92596303e-8f, LN2 = 0.693147181f;
    const float x = -fminf(fmaxf(z, -104.f), 104.f), t = x * L, r = fmaf(x, L_REST, fmaf(x, L, -t));
    float e, q;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, r * LN2, e);
    asm("rcp.approx.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));      // below 2^-126 too
    return q;
  } else {
    return sigmoid_of(z);
  }
}

struct GatedArgs {
  const void *x, *z, *w, *dy;      // z may be null
  long long sx, sz, sdy;           // elements between rows
  void *y, *dx, *dz;               // packed rows
  float *rstd;                     // [rows][groups]; may be null in the forward
  float *part;                     // [blocks][width]; null: not wanted
  long long rows;
  int width, group;
  float eps;
  int gate_first;
};

template <typename T, int TPR, int VPT, bool VEC, bool GATE_FIRST>
__global__ void __launch_bounds__(rv_block<TPR>()) gated_norm_fwd(const GatedArgs a) {
  constexpr int N = RowVec<T>::N, RPB = rv_block<TPR>() / TPR;
  __shared__ float red[2 * (TPR > 32 ? TPR / 32 : 1)];
  const int t = threadIdx.x % TPR, g0 = blockIdx.y * a.group;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  const int G = row < a.rows ? a.group : 0;
  const bool has_z = a.z != nullptr;
  uint4 xv[VPT], zv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    xv[i] = rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.x) + row * a.sx + g0, t, i, G);
    zv[i] = rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.z) + row * a.sz + g0, t, i, has_z ? G : 0);
  }
  float ss[1] = {0.f};
  float gated[GATE_FIRST ? VPT : 1][N];                    // x a(z): the sigmoids are not formed twice
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float x[N];
    rv_unpack<T>(xv[i], x);
    if constexpr (GATE_FIRST) {
      float z[N];
      rv_unpack<T>(zv[i], z);
#pragma unroll
      for (int j = 0; j < N; ++j) gated[i][j] = x[j] *= has_z ? z[j] * gate_sigmoid<T>(z[j]) : 1.f;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) ss[0] += x[j] * x[j];
  }
  rv_team_sum<TPR, 1>(ss, red, 0);
  const float r = rsqrtf(ss[0] / a.group + a.eps);
  if (row >= a.rows) return;
  if (t == 0 && a.rstd) a.rstd[row * gridDim.y + blockIdx.y] = r;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float x[N], w[N];
    rv_unpack<T>(rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.w) + g0, t, i, G), w);
    if constexpr (GATE_FIRST) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = gated[i][j] * r * w[j];
    } else {
      float z[N];
      rv_keep_packed(xv[i]);
      rv_unpack<T>(xv[i], x);
      rv_unpack<T>(zv[i], z);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= r * w[j] * (has_z ? z[j] * gate_sigmoid<T>(z[j]) : 1.f);
    }
    rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + g0, t, i, G, rv_pack<T>(x));
  }
}

// What depends on the row's mean waits in registers for it (the normalised value, dn w, and with the gate first the gate and x a'(z)):
// computed twice, the two transcendentals of every element made this kernel instruction bound (433 us at 16384 x 8192 in groups of
// 1024).  The gradient of a gate behind the norm does not depend on the mean and leaves before it.
template <typename T, int TPR, int VPT, bool VEC, bool GATE_FIRST>
__global__ void __launch_bounds__(rv_block<TPR>()) gated_norm_bwd(const GatedArgs a) {
  constexpr int N = RowVec<T>::N, RPB = rv_block<TPR>() / TPR;
  extern __shared__ __align__(16) uint4 dyn[];
  __shared__ float red[2 * (TPR > 32 ? TPR / 32 : 1)];
  __shared__ float scratch[RPB > 1 ? RPB * TPR * VPT * N : 1];
  enum { XX = 0, DY = 1, ZZ = 2 };
  const int t = threadIdx.x % TPR, g0 = blockIdx.y * a.group;
  const bool has_z = a.z != nullptr;
  const float inv_group = 1.f / a.group;
  float acc[VPT][N] = {};
  RowRing<T, TPR, VPT, VEC, rv_stages(TPR, VPT), 3> in;
  in.ops = 3;
  in.width = a.group;
  in.rows = a.rows;
  in.set(XX, reinterpret_cast<const T*>(a.x) + g0, a.sx);
  in.set(DY, reinterpret_cast<const T*>(a.dy) + g0, a.sdy);
  in.set(ZZ, has_z ? reinterpret_cast<const T*>(a.z) + g0 : nullptr, a.sz);
  const long long step = (long long)gridDim.x * RPB;
  in.start(dyn, (long long)blockIdx.x * RPB + threadIdx.x / TPR, step);
  uint4 wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) wv[i] = rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.w) + g0, t, i, a.group);
  auto stat = [&](long long row) { return row < a.rows ? a.rstd[row * gridDim.y + blockIdx.y] : 0.f; };
  float next_r = stat((long long)blockIdx.x * RPB + threadIdx.x / TPR);      // requested a row ahead
  int turn = 0;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += step, turn ^= 1) {
    const long long row = row0 + threadIdx.x / TPR;
    const int G = row < a.rows ? a.group : 0;
    const float r = next_r;
    next_r = stat(row + step);
    in.wait();
#pragma unroll
    for (int i = 0; i < VPT; ++i) rv_keep_packed(wv[i]);
    float s[1] = {0.f};
    float hat[VPT][N], dnw[VPT][N], gate[GATE_FIRST ? VPT : 1][N], xs[GATE_FIRST ? VPT : 1][N];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float x[N], z[N], d[N], w[N];
      rv_unpack<T>(in.get(XX, i), x);
      rv_unpack<T>(in.get(ZZ, i), z);
      rv_unpack<T>(in.get(DY, i), d);
      rv_unpack<T>(wv[i], w);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float q = gate_sigmoid<T>(z[j]), g = has_z ? z[j] * q : 1.f, slope = q + g * (1.f - q);    // without z no slope is used
        if constexpr (GATE_FIRST) {
          gate[i][j] = g;
          xs[i][j] = x[j] * slope;
          hat[i][j] = x[j] * g * r;
          dnw[i][j] = d[j] * w[j];
          acc[i][j] += d[j] * hat[i][j];
        } else {
          hat[i][j] = x[j] * r;
          const float dh = d[j] * hat[i][j];
          acc[i][j] += dh * g;
          dnw[i][j] = d[j] * g * w[j];
          z[j] = dh * w[j] * slope;
        }
        s[0] += dnw[i][j] * hat[i][j];
      }
      if constexpr (!GATE_FIRST)
        if (a.dz) rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dz) + row * a.width + g0, t, i, G, rv_pack<T>(z));
    }
    in.next();
    rv_team_sum<TPR, 1>(s, red, turn);
    const float m = s[0] * inv_group;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float x[N];
      if constexpr (GATE_FIRST) {
        float z[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float du = r * (dnw[i][j] - hat[i][j] * m);
          x[j] = du * gate[i][j];
          z[j] = du * xs[i][j];
        }
        if (a.dz) rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dz) + row * a.width + g0, t, i, G, rv_pack<T>(z));
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = r * (dnw[i][j] - hat[i][j] * m);
      }
      rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dx) + row * a.width + g0, t, i, G, rv_pack<T>(x));
    }
  }
  in.drain();
  if (a.part) rv_partial<T, TPR, VPT, VEC>(acc, a.part + (long long)blockIdx.x * a.width + g0, a.group, scratch);
}

template <typename T>
static int gated_launch(const GatedArgs& a, bool back, int& blocks, cudaStream_t s) {
  const int size = sizeof(T), nvec = (a.group + RowVec<T>::N - 1) / RowVec<T>::N, groups = a.width / a.group;
  auto fits = [&](const void* p, long long pitch) { return !p || ((reinterpret_cast<uintptr_t>(p) | (pitch * size)) & 15) == 0; };
  const bool vec = a.group * size % 16 == 0 && fits(a.x, a.sx) && fits(a.z, a.sz) && fits(a.w, 0) && fits(a.dy, a.sdy) &&
                   fits(a.y, a.width) && fits(a.dx, a.width) && fits(a.dz, a.width);
  const int team = rv_team(nvec, vec, !back);
#define CM_GATED(TPR, VPT, VEC)                                                                                                  \
  [&] {                                                                                                                          \
    constexpr int TB = rv_block<TPR>(), RPB = TB / TPR;                                                                          \
    if (back) {                                                                                                                  \
      auto kern = a.gate_first ? gated_norm_bwd<T, TPR, VPT, VEC, true> : gated_norm_bwd<T, TPR, VPT, VEC, false>;               \
      constexpr int RING = rv_slots(TPR, VPT, VEC) * VPT * TB * 16 * 3;                                                    \
      static PerDevice configured[2];                                                                                            \
      if (configured[a.gate_first].first()) {                                                                                    \
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING) != cudaSuccess) return -2;             \
        configured[a.gate_first].done();                                                                                         \
      }                                                                                                                          \
      static Resident resident[2];                                                                                                   \
      blocks = rv_blocks(kern, TB, RING, RPB, a.rows, a.width, groups, resident[a.gate_first]);                                                         \
      kern<<<dim3(blocks, groups), TB, RING, s>>>(a);                                                                            \
    } else {                                                                                                                     \
      auto kern = a.gate_first ? gated_norm_fwd<T, TPR, VPT, VEC, true> : gated_norm_fwd<T, TPR, VPT, VEC, false>;               \
      kern<<<dim3(unsigned((a.rows + RPB - 1) / RPB), groups), TB, 0, s>>>(a);                                                   \
    }                                                                                                                            \
    return cudaGetLastError() == cudaSuccess ? 0 : -3;                                                                           \
  }()
  CM_ROW_TEAM(team, vec, CM_GATED);
#undef CM_GATED
}

// `blocks`: out, the partial rows of the backward's weight gradient
static int gated_any(const GatedArgs& a, int dtype, bool back, int& blocks, cudaStream_t s) {
  if (a.group <= 0 || a.width % a.group || a.width / a.group > 65535) return -10;
  switch (dtype) {
    case ROW_BF16: return gated_launch<__nv_bfloat16>(a, back, blocks, s);
    case ROW_FP16: return gated_launch<__half>(a, back, blocks, s);
    case ROW_FP32: return gated_launch<float>(a, back, blocks, s);
  }
  return -10;
}

}  // namespace cm

using namespace cm;

// dtype: 0 bf16, 1 fp16, 2 fp32.  z, rstd may be null; sx, sz: elements between rows; y packed; rstd [rows][width / group].
extern "C" int cm_rmsnorm_gated_fwd(const void* x, long long sx, const void* z, long long sz, const void* w, void* y, float* rstd,
                                    long long rows, int width, int group, int gate_first, float eps, int dtype, cudaStream_t s) {
  if (rows <= 0 || width <= 0) return 0;
  GatedArgs a{};
  a.x = x; a.sx = sx; a.z = z; a.sz = sz; a.w = w; a.y = y; a.rstd = rstd; a.rows = rows; a.width = width; a.group = group;
  a.gate_first = gate_first != 0; a.eps = eps;
  int blocks = 0;
  return gated_any(a, dtype, false, blocks, s);
}

// Partial rows of the weight gradient that the backward needs room for.
extern "C" int cm_rmsnorm_gated_parts(long long rows, int width, int group) {
  return group > 0 ? int(rv_most_blocks(rows, width, width / group)) : 0;
}

// part: [cm_rmsnorm_gated_parts][width] floats of work space, with dw; dz, dw may be null.  dx, dz packed.
extern "C" int cm_rmsnorm_gated_bwd(const void* x, long long sx, const void* z, long long sz, const void* w, const void* dy, long long sdy,
                                    const float* rstd, void* dx, void* dz, void* dw, float* part, long long rows, int width, int group,
                                    int gate_first, int dtype, cudaStream_t s) {
  if (rows <= 0 || width <= 0) return 0;
  GatedArgs a{};
  a.x = x; a.sx = sx; a.z = z; a.sz = sz; a.w = w; a.dy = dy; a.sdy = sdy; a.rstd = const_cast<float*>(rstd); a.dx = dx; a.dz = dz;
  a.part = dw ? part : nullptr; a.rows = rows; a.width = width; a.group = group; a.gate_first = gate_first != 0;
  int blocks = 0;
  const int rc = gated_any(a, dtype, true, blocks, s);
  if (rc || !dw) return rc;
  ColumnSums c{};
  c.partial[0] = part;
  c.out[0] = dw;
  const dim3 grid((width + 31) / 32, 1);
  if (dtype == ROW_BF16) rv_column_sum<__nv_bfloat16><<<grid, 1024, 0, s>>>(c, blocks, width);
  else if (dtype == ROW_FP16) rv_column_sum<__half><<<grid, 1024, 0, s>>>(c, blocks, width);
  else rv_column_sum<float><<<grid, 1024, 0, s>>>(c, blocks, width);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
