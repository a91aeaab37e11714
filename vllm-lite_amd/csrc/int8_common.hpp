// The int8 cache (pa.h): codes int8, K [NB, Hkv, 16, D], V [NB, Hkv, D, 16], and a
// scale byte for each (block, kv head) of each; a value is code * 2^(byte - 127).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pa_common.hpp"

namespace pa {

// Head dims with kernels.
inline bool int8_head_dim(int d) {
  return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256;
}

// 2^(byte - 127) as a float: exact for the bytes 1 to 254 that a scale may have
// (0, in a block never written, gives 0).
__device__ inline float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

}  // namespace pa
