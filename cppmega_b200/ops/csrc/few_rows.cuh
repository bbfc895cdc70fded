// Products of a weight matrix with few rows of activations (`few_rows.cu`): launch interface used by `gated_mlp.cu`.
#pragma once
#include "common.cuh"

namespace cm {
namespace few {

constexpr int MAX_ROWS = 64;        // rows of activations
constexpr int TILE = 128;           // weight rows of a tile

// One product [tokens, N] = X [tokens, K] W [N, K]^T, cut into equal runs of 64-deep k blocks: block c of the grid works on the k blocks
// [c q, (c + 1) q) of the sequence "tile 0's k blocks, tile 1's, ...", and leaves one fp32 partial tile [tokens][128] per weight tile
// that its run touches.  Tile t then is the sum of the partial tiles of the blocks first(t) .. last(t).
struct Cut {
  int tokens, nkb, q, grid, maxseg;
  // 32-bit arithmetic: cut_for refuses more than 2^31 k blocks
  __host__ __device__ int first(int t) const { return int(unsigned(t) * unsigned(nkb) / unsigned(q)); }
  __host__ __device__ int last(int t) const { return int((unsigned(t) * unsigned(nkb) + unsigned(nkb - 1)) / unsigned(q)); }
  // partial tile of weight tile t that block c wrote
  __host__ __device__ long long at(int c, int t) const {
    return ((long long)c * maxseg + (t - int(unsigned(c) * unsigned(q) / unsigned(nkb)))) * tokens * TILE;
  }
  __host__ long long floats() const { return (long long)grid * maxseg * tokens * TILE; }
};
// grid 0: too many k blocks
Cut cut_for(int tokens, int N, int K);

// Programmatic dependent launch: a kernel launched with launch_early may start while its predecessor in the stream still runs, sets
// itself up, and waits in wait_for_input() until all of the predecessor's writes are there.  Everything it reads of the predecessor, and
// everything it overwrites, comes after that wait.  The predecessor's let_next_start() says when it has no more blocks to place.
__device__ __forceinline__ void wait_for_input() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
inline int launch_early(void (*kern)(P...), dim3 grid, dim3 block, int smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P(args)...) == cudaSuccess ? 0 : -3;
}

// X: row pitch ldx; X2: null, or what X lacks (X + X2 is multiplied; same pitch); W: dense rows of K.  Bases and pitches on 16 bytes,
// K % 8 == 0, tokens <= MAX_ROWS.  early: X, and the work space's last reader, are those of the kernel before it in the stream, and the
// weights are older: their loads start before that one has ended.
int launch_partials(const void* X, const void* X2, long long ldx, const void* W, float* part, const Cut& cut, int N, int K, bool early, int* err,
                    cudaStream_t stream);

}  // namespace few
}  // namespace cm
