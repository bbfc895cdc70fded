// Two fp32 values that one instruction works on (fma.rn.f32x2), and the logistic function of one and of two values.
#pragma once
#include "common.cuh"

namespace cm {

struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pr(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ Pair pr(float both) { return pr(both, both); }
__device__ __forceinline__ float2 pr_get(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ float pr_sum(Pair p) {
  const float2 f = pr_get(p);
  return f.x + f.y;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair pr_fma(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

// 1 / (1 + 2^x): the approximations' error is a few 2^-24, and 1 / (1 + inf) is 0, as it should be
__device__ __forceinline__ float logistic2(float x) {
  float e, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));
  return q;
}
// 1 / (1 + exp(-z)); the rounding of z log2(e) adds |z| 2^-24
__device__ __forceinline__ float sigmoid_of(float z) { return logistic2(z * -1.4426950408889634f); }
__device__ __forceinline__ Pair sigmoid_of(Pair z) {
  const float2 x = pr_get(z * pr(-1.4426950408889634f));
  return pr(logistic2(x.x), logistic2(x.y));
}

}  // namespace cm
