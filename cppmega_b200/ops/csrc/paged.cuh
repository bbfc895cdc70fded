// What the kernels of a paged key-value cache share.
#pragma once
#include "common.cuh"

namespace cm {
namespace paged {

// 2^(byte - 127) of an exponent byte; 0 is 2^-127, a subnormal, and 255 infinity
__device__ __forceinline__ float power_of(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }

}  // namespace paged
}  // namespace cm
