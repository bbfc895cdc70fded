// The residual step of a layer with the norms on both sides of the block, forward and backward, in bf16, fp16 or fp32:
//   p = rms(y) post   (or y)            rms(v) = v * rsqrt(mean(v^2) + eps)
//   h = residual + scale * gate * p     gate: none, one per channel, or one per element; rounded to the stream's type
//   n = rms(h) weight                   of the rounded h: what the stream holds is what is normalised
// Backward, with a = scale * gate * post, r and rho the two reciprocal norms, yh = y r, hh = h rho, and dh0 the gradient that reaches h
// from its other readers:
//   g = dn weight;  dh = rho (g - hh mean(g hh)) + dh0;  dresidual = dh;  dweight = sum dn hh
//   dp = scale gate dh;  dgate = scale dh p;  dpost = sum dp yh;  dy = r (a dh - yh mean(a dh yh))
// The second mean is linear in the first: with S1 = sum g hh, S2 = sum a yh (rho g + dh0), S3 = sum a yh hh it is
// (S2 - rho S1 S3 / W) / W, so that a row is read once and reduced once.
// Bound by memory: forward 4 rows moved, backward 4, with post norm or gate 6.  16384 x 4096 in bf16: forward 80 us and backward 94 (83 each
// at the copy rate); with post norm and gate 88 and 162 (83, 125): two blocks an SM, for its 128 registers, do not hide the time between a
// row's sums and its results.  A team of threads holds a row (rv_team), so that it crosses memory once each way.  Sums over rows go through
// one partial row per block and a second kernel in a fixed order: the same call gives the same bits.
#include "row_vec.cuh"
#define CM_ROW_TEAM_BY_WARP(team, F)

namespace cm {

struct ResidualArgs {
  const void *y, *res, *w, *post, *gate;      // post, gate may be null
  long long sy, sres;                         // elements between rows
  int gate_rows;                              // gate: 0 one per channel, 1 one per element (packed rows)
  void *n, *h;
  float *rstd_y, *rstd_h;                     // may be null
  long long rows;
  int width;
  float scale, eps;
  // backward
  const void *dn, *dh;                        // either may be null: zero
  long long sdn, sdh;
  void *dres, *dy, *dgate_rows;               // dy null: the same as dres
  float *part_w, *part_post, *part_gate;      // [blocks][width]; null: not wanted
  int ring_ops;                               // operands in the ring
};

template <typename T, int TPR, int VPT, bool VEC, bool FULL>
__global__ void __launch_bounds__(rv_block<TPR>()) residual_norm_fwd(const ResidualArgs a) {
  constexpr int H = RowVec<T>::N / 2, RPB = rv_block<TPR>() / TPR;
  __shared__ float red[2 * (TPR > 32 ? TPR / 32 : 1)];
  const int t = threadIdx.x % TPR, W = a.width;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool on = row < a.rows;
  const int w_on = on ? W : 0;                // a team past the last row reads and writes nothing but takes part in the sums
  const T* yr = reinterpret_cast<const T*>(a.y) + row * a.sy;
  const T* xr = reinterpret_cast<const T*>(a.res) + row * a.sres;
  uint4 yv[VPT], hv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    yv[i] = rv_load<T, TPR, VEC>(yr, t, i, w_on);
    hv[i] = rv_load<T, TPR, VEC>(xr, t, i, w_on);
  }
  float r = 1.f;
  const bool post = FULL && a.post;
  if (post) {
    Pair sq = {};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      Pair f[H];
      rv_unpack<T>(yv[i], f);
#pragma unroll
      for (int j = 0; j < H; ++j) sq = pr_fma(f[j], f[j], sq);
    }
    float ss[1] = {pr_sum(sq)};
    rv_team_sum<TPR, 1>(ss, red, 0);
    r = rsqrtf(ss[0] / W + a.eps);
    if (on && t == 0 && a.rstd_y) a.rstd_y[row] = r;
  }
  Pair sq = {};
  const Pair sr = pr(a.scale * r);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    Pair y[H], x[H];
    rv_unpack<T>(yv[i], y);
    rv_unpack<T>(hv[i], x);
    if constexpr (FULL) {
      if (post) {
        Pair p[H];
        rv_unpack<T>(rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.post), t, i, W), p);
#pragma unroll
        for (int j = 0; j < H; ++j) y[j] = y[j] * p[j];
      }
      if (a.gate) {
        Pair g[H];
        rv_unpack<T>(rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.gate) + (a.gate_rows ? row * W : 0ll), t, i, w_on), g);
#pragma unroll
        for (int j = 0; j < H; ++j) y[j] = y[j] * g[j];
      }
    }
#pragma unroll
    for (int j = 0; j < H; ++j) x[j] = pr_fma(sr, y[j], x[j]);
    hv[i] = rv_pack<T>(x);
    rv_unpack<T>(hv[i], x);                   // the stream's value
#pragma unroll
    for (int j = 0; j < H; ++j) sq = pr_fma(x[j], x[j], sq);
  }
  float ss[1] = {pr_sum(sq)};
  rv_team_sum<TPR, 1>(ss, red, 1);
  const float rho = rsqrtf(ss[0] / W + a.eps);
  if (!on) return;
  if (t == 0 && a.rstd_h) a.rstd_h[row] = rho;
  T* hr = reinterpret_cast<T*>(a.h) + row * W;
  T* nr = reinterpret_cast<T*>(a.n) + row * W;
  const Pair rho2 = pr(rho);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    Pair x[H], w[H];
    rv_unpack<T>(hv[i], x);
    rv_unpack<T>(rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.w), t, i, W), w);
    rv_store<T, TPR, VEC>(hr, t, i, W, hv[i]);
#pragma unroll
    for (int j = 0; j < H; ++j) x[j] = x[j] * rho2 * w[j];
    rv_store<T, TPR, VEC>(nr, t, i, W, rv_pack<T>(x));
  }
}

template <typename T, int TPR, int VPT, bool VEC, bool FULL>
__global__ void __launch_bounds__(rv_block<TPR>(), rv_block<TPR>() >= 512 ? 1 : (FULL ? 512 : 768) / rv_block<TPR>()) residual_norm_bwd(const ResidualArgs a) {
  constexpr int N = RowVec<T>::N, H = N / 2, RPB = rv_block<TPR>() / TPR;
  extern __shared__ __align__(16) uint4 dyn[];
  __shared__ float red[2 * (FULL ? 3 : 1) * (TPR > 32 ? TPR / 32 : 1)];
  __shared__ float scratch[RPB > 1 ? RPB * TPR * VPT * N : 1];
  enum { HH = 0, DN = 1, DH = 2, YY = 3, GG = 4 };
  const int t = threadIdx.x % TPR, W = a.width;
  Pair acc_w[VPT][H] = {}, acc_y[FULL ? VPT : 1][H] = {};
  const bool post = FULL && a.post, gate = FULL && a.gate;
  RowRing<T, TPR, VPT, VEC, rv_stages(TPR, VPT), FULL ? 5 : 3> in;
  in.ops = a.ring_ops;
  in.width = W;
  in.rows = a.rows;
  in.set(DN, a.dn, a.sdn);
  in.set(DH, a.dh, a.sdh);
  in.set(HH, a.h, W);
  if constexpr (FULL) {
    in.set(YY, a.y, a.sy);
    in.set(GG, a.gate_rows ? a.gate : nullptr, W);
  }
  const long long step = (long long)gridDim.x * RPB, first = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  in.start(dyn, first, step);
  // the parameters of this thread's columns, as they come; a missing post norm or gate is a factor of one
  uint4 wv[VPT], pv[FULL ? VPT : 1], tv[FULL ? VPT : 1];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    wv[i] = rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.w), t, i, W);
    if constexpr (FULL) {
      pv[i] = post ? rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.post), t, i, W) : rv_ones<T>();
      tv[i] = gate && !a.gate_rows ? rv_load<T, TPR, VEC>(reinterpret_cast<const T*>(a.gate), t, i, W) : rv_ones<T>();
    }
  }
  const float inv_w = 1.f / W;
  float next_rho, next_r;                                   // of the next row, requested a row ahead
  auto stats = [&](long long row) {
    next_rho = row < a.rows ? a.rstd_h[row] : 0.f;
    next_r = !post ? 1.f : row < a.rows ? a.rstd_y[row] : 0.f;
  };
  stats(first);
  int turn = 0;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += step, turn ^= 1) {
    const long long row = row0 + threadIdx.x / TPR;
    const bool on = row < a.rows;
    const float rho = next_rho, r = next_r;
    stats(row + step);
    in.wait();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      rv_keep_packed(wv[i]);
      if constexpr (FULL) {
        rv_keep_packed(pv[i]);
        rv_keep_packed(tv[i]);
      }
    }
    // s[0] = sum g h, s[1] = sum gate post y (rho g + dh0), s[2] = sum gate post y h: the constant factors follow behind the sums
    Pair sp[FULL ? 3 : 1] = {};
    Pair dt[VPT][H];                                        // rho g + dh0
    const Pair rho2 = pr(rho);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      Pair g[H], h[H], w[H];
      rv_unpack<T>(in.get(DN, i), g);
      rv_unpack<T>(in.get(HH, i), h);
      rv_unpack<T>(in.get(DH, i), dt[i]);
      rv_unpack<T>(wv[i], w);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        acc_w[i][j] = pr_fma(g[j], h[j] * rho2, acc_w[i][j]);
        g[j] = g[j] * w[j];
        sp[0] = pr_fma(g[j], h[j], sp[0]);
        dt[i][j] = pr_fma(rho2, g[j], dt[i][j]);
      }
      if constexpr (FULL) {
        Pair y[H], p[H], q[H];
        rv_unpack<T>(in.get(YY, i), y);
        rv_unpack<T>(pv[i], p);
        rv_unpack<T>(a.gate_rows ? in.get(GG, i) : tv[i], q);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const Pair ay = p[j] * q[j] * y[j];
          sp[1] = pr_fma(ay, dt[i][j], sp[1]);
          sp[2] = pr_fma(ay, h[j], sp[2]);
        }
      }
    }
    float s[FULL ? 3 : 1];
#pragma unroll
    for (int k = 0; k < (FULL ? 3 : 1); ++k) s[k] = pr_sum(sp[k]);
    rv_team_sum<TPR, FULL ? 3 : 1>(s, red, turn);
    const float k = rho * s[0] * inv_w * rho * rho;         // dh = rho g + dh0 - k h; rho^3 alone may underflow
    float m2 = 0.f;                                         // mean(gate post dh yh)
    if constexpr (FULL) m2 = post ? r * (s[1] - k * s[2]) * inv_w : 0.f;
    const Pair k2 = pr(-k), r2 = pr(r), sr2 = pr(a.scale * r), m22 = pr(-m2), scale2 = pr(a.scale);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      Pair d[H];
      rv_unpack<T>(in.get(HH, i), d);
#pragma unroll
      for (int j = 0; j < H; ++j) d[j] = pr_fma(k2, d[j], dt[i][j]);
      rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dres) + row * W, t, i, on ? W : 0, rv_pack<T>(d));
      if constexpr (FULL) {
        Pair y[H], p[H], q[H];
        rv_unpack<T>(in.get(YY, i), y);
        rv_unpack<T>(pv[i], p);
        if (a.gate_rows) {
          rv_unpack<T>(in.get(GG, i), q);
          if (a.dgate_rows) {
            Pair dg[H];
#pragma unroll
            for (int j = 0; j < H; ++j) dg[j] = sr2 * d[j] * (y[j] * p[j]);
            rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dgate_rows) + row * W, t, i, on ? W : 0, rv_pack<T>(dg));
          }
#pragma unroll
          for (int j = 0; j < H; ++j) {
            y[j] = y[j] * r2;
            d[j] = d[j] * q[j];
            acc_y[i][j] = pr_fma(d[j], y[j], acc_y[i][j]);
          }
        } else {
          rv_unpack<T>(tv[i], q);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            y[j] = y[j] * r2;
            acc_y[i][j] = pr_fma(d[j], y[j], acc_y[i][j]);
            d[j] = d[j] * q[j];
          }
        }
#pragma unroll
        for (int j = 0; j < H; ++j) d[j] = sr2 * pr_fma(m22, y[j], d[j] * p[j]);
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) d[j] = d[j] * scale2;
      }
      if (a.dy) rv_store<T, TPR, VEC>(reinterpret_cast<T*>(a.dy) + row * W, t, i, on ? W : 0, rv_pack<T>(d));
    }
    in.next();
  }
  in.drain();
  const long long at = (long long)blockIdx.x * W;
  if (a.part_w) rv_partial<T, TPR, VPT, VEC>(acc_w, a.part_w + at, W, scratch);
  if constexpr (FULL) {
    // with a gate per channel both its gradient and the post norm's are the sum of dh yh, times the other one's factor; with a gate per
    // element the sum already holds the gate
    auto out = [&](float* part, const uint4 (&factor)[VPT]) {
      Pair sum[VPT][H];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        rv_unpack<T>(factor[i], sum[i]);
#pragma unroll
        for (int j = 0; j < H; ++j) sum[i][j] = pr(a.scale) * sum[i][j] * acc_y[i][j];
      }
      rv_partial<T, TPR, VPT, VEC>(sum, part + at, W, scratch);
    };
    if (a.part_post) out(a.part_post, tv);
    if (a.part_gate) out(a.part_gate, pv);
  }
}

static bool aligned16(const void* p, long long pitch, int size) { return !p || ((reinterpret_cast<uintptr_t>(p) | (pitch * size)) & 15) == 0; }

static bool residual_vec(const ResidualArgs& a, int size) {
  const long long W = a.width;
  return (W * size) % 16 == 0 && aligned16(a.y, a.sy, size) && aligned16(a.res, a.sres, size) && aligned16(a.w, 0, size) &&
         aligned16(a.post, 0, size) && aligned16(a.gate, 0, size) && aligned16(a.n, 0, size) && aligned16(a.h, 0, size) &&
         aligned16(a.dn, a.sdn, size) && aligned16(a.dh, a.sdh, size) && aligned16(a.dres, 0, size) && aligned16(a.dy, 0, size) &&
         aligned16(a.dgate_rows, 0, size);
}

template <typename T, bool FULL>
static int residual_launch(const ResidualArgs& a, bool back, int& blocks, cudaStream_t s) {
  const int size = sizeof(T), nvec = (a.width + RowVec<T>::N - 1) / RowVec<T>::N;
  const bool vec = residual_vec(a, size);
  const int team = rv_team(nvec, vec, false);
#define CM_RES(TPR, VPT, VEC)                                                                                                     \
  [&] {                                                                                                                           \
    constexpr int TB = rv_block<TPR>(), RPB = TB / TPR;                                                                           \
    if (back) {                                                                                                                   \
      auto kern = residual_norm_bwd<T, TPR, VPT, VEC, FULL>;                                                                      \
      constexpr int SLOT = rv_slots(TPR, VPT, VEC) * VPT * TB * 16;                                                         \
      static PerDevice configured;                                                                                                \
      if (configured.first()) {                                                                                                   \
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SLOT * (FULL ? 5 : 3)) != cudaSuccess) return -2; \
        configured.done();                                                                                                        \
      }                                                                                                                           \
      static Resident resident[6];                                                                                                    \
      blocks = rv_blocks(kern, TB, SLOT * a.ring_ops, RPB, a.rows, a.width, 1, resident[a.ring_ops]);                                    \
      kern<<<blocks, TB, SLOT * a.ring_ops, s>>>(a);                                                                              \
    } else residual_norm_fwd<T, TPR, VPT, VEC, FULL><<<unsigned((a.rows + RPB - 1) / RPB), TB, 0, s>>>(a);                          \
    return cudaGetLastError() == cudaSuccess ? 0 : -3;                                                                            \
  }()
  CM_ROW_TEAM(team, vec, CM_RES);
#undef CM_RES
}

// `blocks`: out, the partial rows of a backward's column sums
static int residual_any(const ResidualArgs& a, int dtype, bool back, int& blocks, cudaStream_t s) {
  const bool full = a.post || a.gate;
  switch (dtype) {
    case ROW_BF16: return full ? residual_launch<__nv_bfloat16, true>(a, back, blocks, s) : residual_launch<__nv_bfloat16, false>(a, back, blocks, s);
    case ROW_FP16: return full ? residual_launch<__half, true>(a, back, blocks, s) : residual_launch<__half, false>(a, back, blocks, s);
    case ROW_FP32: return full ? residual_launch<float, true>(a, back, blocks, s) : residual_launch<float, false>(a, back, blocks, s);
  }
  return -10;
}

}  // namespace cm

using namespace cm;

// dtype: 0 bf16, 1 fp16, 2 fp32 (all tensors; the statistics are fp32).  post / gate / rstd_* may be null.  sy, sres: elements between
// rows; gate_rows: the gate has a row per row of y.
extern "C" int cm_residual_rmsnorm_fwd(const void* y, long long sy, const void* res, long long sres, const void* w, const void* post,
                                       const void* gate, int gate_rows, void* n, void* h, float* rstd_y, float* rstd_h, long long rows,
                                       int width, float scale, float eps, int dtype, cudaStream_t s) {
  if (rows <= 0 || width <= 0) return 0;
  ResidualArgs a{};
  a.y = y; a.sy = sy; a.res = res; a.sres = sres; a.w = w; a.post = post; a.gate = gate; a.gate_rows = gate_rows;
  a.n = n; a.h = h; a.rstd_y = rstd_y; a.rstd_h = rstd_h; a.rows = rows; a.width = width; a.scale = scale; a.eps = eps;
  int blocks = 0;
  return residual_any(a, dtype, false, blocks, s);
}

// Partial rows of a column sum that the backward needs room for.
extern "C" int cm_residual_rmsnorm_parts(long long rows, int width) { return int(rv_most_blocks(rows, width, 1)); }

// part: [3][cm_residual_rmsnorm_parts][width] floats of work space.  dn, dh (gradients of n and h) may be null; dy null: it is dres (no post
// norm, no gate, scale 1); dw, dpost, dgate (one per channel), dgate_rows may be null.
extern "C" int cm_residual_rmsnorm_bwd(const void* dn, long long sdn, const void* dh, long long sdh, const void* h, const void* y,
                                       long long sy, const void* w, const void* post, const void* gate, int gate_rows,
                                       const float* rstd_y, const float* rstd_h, void* dres, void* dy, void* dgate_rows, void* dw,
                                       void* dpost, void* dgate, float* part, long long rows, int width, float scale, int dtype,
                                       cudaStream_t s) {
  if (rows <= 0 || width <= 0) return 0;
  ResidualArgs a{};
  a.dn = dn; a.sdn = sdn; a.dh = dh; a.sdh = sdh; a.h = const_cast<void*>(h); a.y = y; a.sy = sy; a.w = w; a.post = post; a.gate = gate;
  a.gate_rows = gate_rows; a.rstd_y = const_cast<float*>(rstd_y); a.rstd_h = const_cast<float*>(rstd_h); a.dres = dres; a.dy = dy;
  a.dgate_rows = dgate_rows; a.rows = rows; a.width = width; a.scale = scale;
  a.ring_ops = !post && !gate ? 3 : gate && gate_rows ? 5 : 4;
  ColumnSums c{};
  int sums = 0;
  auto want = [&](void* out, float*& slot) {
    if (!out) return;
    slot = part + sums * rv_most_blocks(rows, width, 1) * width;
    c.partial[sums] = slot;
    c.out[sums++] = out;
  };
  want(dw, a.part_w);
  want(dpost, a.part_post);
  want(dgate, a.part_gate);
  int blocks = 0;
  const int rc = residual_any(a, dtype, true, blocks, s);
  if (rc || !sums) return rc;
  const dim3 grid((width + 31) / 32, sums);
  if (dtype == ROW_BF16) rv_column_sum<__nv_bfloat16><<<grid, 1024, 0, s>>>(c, blocks, width);
  else if (dtype == ROW_FP16) rv_column_sum<__half><<<grid, 1024, 0, s>>>(c, blocks, width);
  else rv_column_sum<float><<<grid, 1024, 0, s>>>(c, blocks, width);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
