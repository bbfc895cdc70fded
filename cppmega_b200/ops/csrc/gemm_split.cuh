// Dense product with the reduction of its last tiles cut over idle SMs (`gemm_split.cu`): launch interface used by `gated_mlp.cu`.
#pragma once
#include "common.cuh"

namespace cm {
namespace split {

// How C [M, N] is worked on: rows [0, whole) by cm_gemm_bf16, the rest in tiles of 256 x bn whose reduction is cut into `slices` runs of
// `kb_per_slice` 64-deep k blocks.  slices 0: all rows by cm_gemm_bf16.
struct Plan {
  int whole, bn, slices, kb_per_slice;
  long long floats;        // work space: one fp32 copy of the split rows per slice
};
Plan plan(int sms, int M, int N, int K, bool b_mn);     // on a chip of `sms` SMs

// As cm_gemm_bf16; ws: plan(sm_count(), ...).floats floats.
int gemm(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc, bool a_mn, bool b_mn,
         bool out_fp32, bool accumulate, float* ws, int* err, cudaStream_t stream);

}  // namespace split
}  // namespace cm
